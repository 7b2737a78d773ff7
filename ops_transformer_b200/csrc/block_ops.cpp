// Host side of the operators around the expert FFN (include/gmm_b200.h): add_rms_norm_quant, route_top_k, adapter_add, quant_matmul,
// sandwich_norm_quant, expert_balance and its gradient.  The first phase checks and builds the executor; it is host only and never reads a tensor.  Nothing may leave an entry point as an exception.
#include <cmath>
#include <initializer_list>

#include "gmm_b200.h"
#include "op_api.h"

namespace gmm {
namespace {

constexpr int64_t kMaxAxis = 65535;          // as for the inner axes of the grouped GEMM
constexpr int64_t kMaxChannels = 1 << 24;    // of a dense product: a vocabulary
constexpr int64_t kMaxRows = 0x7fffffffll / 2;

// A tensor that may be absent, but not with elements and without an address, nor in a private format.
bool usable(const aclTensor *t) { return !t || ((t->data || t->empty()) && !is_private_format(t->format)); }
bool on_boundary(const aclTensor *t) { return !t || t->empty() || reinterpret_cast<uintptr_t>(tensor_ptr(t)) % dtype_size(t->dtype) == 0; }

bool is_float(aclDataType t) { return t == ACL_FLOAT || t == ACL_FLOAT16 || t == ACL_BF16; }

// An executor that is dropped unless it is handed out.
struct NewExecutor {
    aclOpExecutor *e;
    explicit NewExecutor(const char *name) : e(new_executor(name)) {}
    ~NewExecutor() { delete e; }
    aclnnStatus hand_out(uint64_t *size, aclOpExecutor **out)
    {
        const aclnnStatus rc = finish_phase1(e, size, out);
        e = nullptr;
        return rc;
    }
};

#define REQUIRE_NOT_NULL(t) GMM_REQUIRE((t) != nullptr, ACLNN_ERR_PARAM_NULLPTR, #t " must not be nullptr.")
#define REQUIRE_RANK(t, r) GMM_REQUIRE((t)->rank() == (r), ACLNN_ERR_PARAM_INVALID, #t " dim num should be %d, but now is %zu.", (r), (t)->rank())
#define REQUIRE_USABLE(...)                                                                                                          \
    for (const aclTensor *t_ : std::initializer_list<const aclTensor *>{__VA_ARGS__}) {                                               \
        GMM_REQUIRE(usable(t_), ACLNN_ERR_PARAM_INVALID, "tensors must have an address and must not have a private format.");        \
        GMM_REQUIRE(on_boundary(t_), ACLNN_ERR_PARAM_INVALID, "tensors must be aligned to their elements.");                         \
    }
#define REQUIRE_SHAPE1(t, a) \
    GMM_REQUIRE((t)->rank() == 1 && (t)->dim(0) == (a), ACLNN_ERR_PARAM_INVALID, #t " shape must be [%lld].", (long long)(a))
#define REQUIRE_SHAPE2(t, a, b)                                                                                                     \
    GMM_REQUIRE((t)->rank() == 2 && (t)->dim(0) == (a) && (t)->dim(1) == (b), ACLNN_ERR_PARAM_INVALID, #t " shape must be [%lld, %lld].", \
                (long long)(a), (long long)(b))
#define REQUIRE_SHAPE3(t, a, b, c)                                                                                                    \
    GMM_REQUIRE((t)->rank() == 3 && (t)->dim(0) == (a) && (t)->dim(1) == (b) && (t)->dim(2) == (c), ACLNN_ERR_PARAM_INVALID, \
                #t " shape must be [%lld, %lld, %lld].", (long long)(a), (long long)(b), (long long)(c))

aclnnStatus norm_phase1(const aclTensor *x, const aclTensor *residual, const aclTensor *gamma, const aclTensor *smooth, float eps,
                        aclTensor *q, aclTensor *scale, aclTensor *residualOut, aclTensor *normedOut, uint64_t *workspaceSize,
                        aclOpExecutor **executor)
{
    REQUIRE_NOT_NULL(workspaceSize); REQUIRE_NOT_NULL(executor);
    REQUIRE_NOT_NULL(x); REQUIRE_NOT_NULL(gamma); REQUIRE_NOT_NULL(q); REQUIRE_NOT_NULL(scale);
    GMM_REQUIRE(!residualOut || residual, ACLNN_ERR_PARAM_NULLPTR, "residualOut needs a residual.");
    REQUIRE_RANK(x, 2);
    const int64_t rows = x->dim(0), h = x->dim(1);
    GMM_REQUIRE(is_float(x->dtype), ACLNN_ERR_PARAM_INVALID, "x dtype must be float32, float16 or bfloat16.");
    GMM_REQUIRE(h >= 1 && h <= kMaxAxis, ACLNN_ERR_PARAM_INVALID, "x's rows must have 1 to %lld elements, but have %lld.", (long long)kMaxAxis, (long long)h);
    GMM_REQUIRE(rows >= 0 && rows <= kMaxRows, ACLNN_ERR_PARAM_INVALID, "x must not have more than %lld rows.", (long long)kMaxRows);
    REQUIRE_SHAPE1(gamma, h);
    GMM_REQUIRE(gamma->dtype == x->dtype || gamma->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "gamma dtype must be x's or float32.");
    REQUIRE_SHAPE2(q, rows, h);
    GMM_REQUIRE(q->dtype == ACL_INT8, ACLNN_ERR_PARAM_INVALID, "q dtype must be int8.");
    REQUIRE_SHAPE1(scale, rows);
    GMM_REQUIRE(scale->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "scale dtype must be float32.");
    if (residual) {
        REQUIRE_SHAPE2(residual, rows, h);
        GMM_REQUIRE(residual->dtype == x->dtype, ACLNN_ERR_PARAM_INVALID, "residual dtype must be x's.");
    }
    if (smooth) {
        REQUIRE_SHAPE1(smooth, h);
        GMM_REQUIRE(smooth->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "smooth dtype must be float32.");
    }
    for (const aclTensor *t : {residualOut, normedOut}) {
        if (!t) continue;
        GMM_REQUIRE(t->rank() == 2 && t->dim(0) == rows && t->dim(1) == h && t->dtype == x->dtype, ACLNN_ERR_PARAM_INVALID,
                    "residualOut and normedOut must have x's shape and dtype.");
    }
    REQUIRE_USABLE(x, residual, gamma, smooth, q, scale, residualOut, normedOut);
    GMM_REQUIRE(eps > 0.0f && std::isfinite(eps), ACLNN_ERR_PARAM_INVALID, "eps must be positive and finite.");

    NewExecutor ne("gmmB200AddRmsNormQuant");
    aclOpExecutor *e = ne.e;
    GMM_REQUIRE(e != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "cannot create executor.");
    if (rows > 0) {
        NormQuantProblem &p = e->norm;
        bind_rows(e, x, &p.x, &p.ld_x, false);
        bind_rows(e, residual, &p.residual, &p.ld_residual, false);
        bind_tensor(e, gamma, &p.gamma, false);
        bind_tensor(e, smooth, &p.smooth, false);
        bind_rows(e, q, &p.q, &p.ld_q, true);
        bind_tensor(e, scale, &p.scale, true);
        bind_rows(e, residualOut, &p.residual_out, &p.ld_residual_out, true);
        bind_rows(e, normedOut, &p.normed_out, &p.ld_normed, true);
        p.rows = rows; p.h = h;
        p.dtype = (int)x->dtype; p.gamma_dtype = (int)gamma->dtype;
        p.eps = eps;
        e->kind = aclOpExecutor::kNormQuant;
    }
    return ne.hand_out(workspaceSize, executor);
}

aclnnStatus route_phase1(const aclTensor *logits, const aclTensor *bias, const aclTensor *tokenMask, int64_t scoring, int64_t nGroup,
                         int64_t topkGroup, int64_t groupScore, bool renormalize, float scale, aclTensor *weights, aclTensor *ids,
                         uint64_t *workspaceSize, aclOpExecutor **executor)
{
    REQUIRE_NOT_NULL(workspaceSize); REQUIRE_NOT_NULL(executor);
    REQUIRE_NOT_NULL(logits); REQUIRE_NOT_NULL(weights); REQUIRE_NOT_NULL(ids);
    REQUIRE_RANK(logits, 2); REQUIRE_RANK(weights, 2); REQUIRE_RANK(ids, 2);
    const int64_t rows = logits->dim(0), experts = logits->dim(1), k = weights->dim(1);
    GMM_REQUIRE(is_float(logits->dtype), ACLNN_ERR_PARAM_INVALID, "logits dtype must be float32, float16 or bfloat16.");
    GMM_REQUIRE(experts >= 1 && experts <= 1024, ACLNN_ERR_PARAM_INVALID, "logits must name 1 to 1024 experts, but name %lld.", (long long)experts);
    GMM_REQUIRE(rows >= 0 && rows <= kMaxRows, ACLNN_ERR_PARAM_INVALID, "logits must not have more than %lld rows.", (long long)kMaxRows);
    GMM_REQUIRE(scoring == kScoreSoftmax || scoring == kScoreSigmoid, ACLNN_ERR_PARAM_INVALID, "scoring must be 0 (softmax) or 1 (sigmoid).");
    GMM_REQUIRE(groupScore == kGroupMax || groupScore == kGroupTop2, ACLNN_ERR_PARAM_INVALID, "groupScore must be 0 (largest) or 1 (sum of the two largest).");
    GMM_REQUIRE(nGroup >= 1 && nGroup <= 32 && experts % nGroup == 0, ACLNN_ERR_PARAM_INVALID,
                "nGroup must be in [1, 32] and divide the %lld experts, but is %lld.", (long long)experts, (long long)nGroup);
    GMM_REQUIRE(topkGroup >= 1 && topkGroup <= nGroup, ACLNN_ERR_PARAM_INVALID, "topkGroup must be in [1, nGroup], but is %lld.", (long long)topkGroup);
    GMM_REQUIRE(k >= 1 && k <= 32 && k <= topkGroup * (experts / nGroup), ACLNN_ERR_PARAM_INVALID,
                "top_k must be in [1, 32] and at most the %lld experts of the chosen groups, but is %lld.",
                (long long)(topkGroup * (experts / nGroup)), (long long)k);
    GMM_REQUIRE(std::isfinite(scale), ACLNN_ERR_PARAM_INVALID, "scale must be finite.");
    REQUIRE_SHAPE2(weights, rows, k); REQUIRE_SHAPE2(ids, rows, k);
    GMM_REQUIRE(weights->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "weights dtype must be float32.");
    GMM_REQUIRE(ids->dtype == ACL_INT32 || ids->dtype == ACL_INT64, ACLNN_ERR_PARAM_INVALID, "ids dtype must be int32 or int64.");
    if (bias) {
        REQUIRE_SHAPE1(bias, experts);
        GMM_REQUIRE(bias->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "bias dtype must be float32.");
    }
    if (tokenMask) {
        REQUIRE_SHAPE1(tokenMask, rows);
        GMM_REQUIRE(tokenMask->dtype == ACL_INT8 || tokenMask->dtype == ACL_BOOL, ACLNN_ERR_PARAM_INVALID, "tokenMask dtype must be int8 or bool.");
    }
    REQUIRE_USABLE(logits, bias, tokenMask, weights, ids);

    NewExecutor ne("gmmB200RouteTopK");
    aclOpExecutor *e = ne.e;
    GMM_REQUIRE(e != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "cannot create executor.");
    if (rows > 0) {
        RouteTopKProblem &p = e->route;
        bind_rows(e, logits, &p.logits, &p.ld, false);
        p.dtype = (int)logits->dtype;
        bind_tensor(e, bias, &p.bias, false);
        bind_tensor(e, tokenMask, &p.token_mask, false);
        bind_tensor(e, weights, &p.weights, true);
        bind_tensor(e, ids, &p.ids, true);
        p.ids_i64 = ids->dtype == ACL_INT64;
        p.rows = rows; p.experts = (int)experts; p.top_k = (int)k;
        p.scoring = (int)scoring; p.group_score = (int)groupScore;
        p.n_group = (int)nGroup; p.topk_group = (int)topkGroup;
        p.renormalize = renormalize; p.scale = scale;
        e->kind = aclOpExecutor::kRouteTopK;
    }
    return ne.hand_out(workspaceSize, executor);
}

aclnnStatus adapter_phase1(const aclTensor *base, const aclTensor *x, const aclTensor *xScale, const aclTensor *a, const aclTensor *b,
                           const aclTensor *adapterIds, const aclTensor *scaling, aclTensor *out, uint64_t *workspaceSize,
                           aclOpExecutor **executor)
{
    REQUIRE_NOT_NULL(workspaceSize); REQUIRE_NOT_NULL(executor);
    REQUIRE_NOT_NULL(base); REQUIRE_NOT_NULL(x); REQUIRE_NOT_NULL(a); REQUIRE_NOT_NULL(b); REQUIRE_NOT_NULL(adapterIds); REQUIRE_NOT_NULL(out);
    REQUIRE_RANK(base, 2); REQUIRE_RANK(x, 2); REQUIRE_RANK(a, 3);
    const int64_t rows = base->dim(0), n = base->dim(1), k = x->dim(1), adapters = a->dim(0), rank = a->dim(1);
    GMM_REQUIRE(base->dtype == ACL_FLOAT16 || base->dtype == ACL_BF16, ACLNN_ERR_PARAM_INVALID, "base dtype must be float16 or bfloat16.");
    GMM_REQUIRE(rows >= 0 && rows <= kMaxRows, ACLNN_ERR_PARAM_INVALID, "base must not have more than %lld rows.", (long long)kMaxRows);
    GMM_REQUIRE(n >= 1 && n <= kMaxAxis && k >= 1 && k <= kMaxAxis, ACLNN_ERR_PARAM_INVALID, "k and n must be in [1, %lld].", (long long)kMaxAxis);
    GMM_REQUIRE(rank >= 1 && rank <= 128, ACLNN_ERR_PARAM_INVALID, "rank must be in [1, 128], but is %lld.", (long long)rank);
    GMM_REQUIRE(adapters >= 1 && adapters <= 16384, ACLNN_ERR_PARAM_INVALID, "a must hold 1 to 16384 adapters, but holds %lld.", (long long)adapters);
    REQUIRE_SHAPE2(x, rows, k);
    GMM_REQUIRE(x->dtype == base->dtype || x->dtype == ACL_INT8, ACLNN_ERR_PARAM_INVALID, "x dtype must be base's or int8.");
    GMM_REQUIRE(x->dtype != ACL_INT8 || xScale, ACLNN_ERR_PARAM_NULLPTR, "an int8 x needs xScale.");
    GMM_REQUIRE(x->dtype == ACL_INT8 || !xScale, ACLNN_ERR_PARAM_INVALID, "xScale belongs to an int8 x.");
    REQUIRE_SHAPE3(a, adapters, rank, k); REQUIRE_SHAPE3(b, adapters, n, rank);
    GMM_REQUIRE(a->dtype == base->dtype && b->dtype == base->dtype, ACLNN_ERR_PARAM_INVALID, "a and b must have base's dtype.");
    REQUIRE_SHAPE1(adapterIds, rows);
    GMM_REQUIRE(adapterIds->dtype == ACL_INT32, ACLNN_ERR_PARAM_INVALID, "adapterIds dtype must be int32.");
    REQUIRE_SHAPE2(out, rows, n);
    GMM_REQUIRE(out->dtype == base->dtype, ACLNN_ERR_PARAM_INVALID, "out dtype must be base's.");
    if (xScale) {
        REQUIRE_SHAPE1(xScale, rows);
        GMM_REQUIRE(xScale->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "xScale dtype must be float32.");
    }
    if (scaling) {
        REQUIRE_SHAPE1(scaling, adapters);
        GMM_REQUIRE(scaling->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "scaling dtype must be float32.");
    }
    REQUIRE_USABLE(base, x, xScale, a, b, adapterIds, scaling, out);

    NewExecutor ne("gmmB200AdapterAdd");
    aclOpExecutor *e = ne.e;
    GMM_REQUIRE(e != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "cannot create executor.");
    if (rows > 0) {
        AdapterProblem &p = e->adapter;
        bind_rows(e, base, &p.base, &p.ld_base, false);
        bind_rows(e, x, &p.x, &p.ld_x, false);
        bind_tensor(e, xScale, &p.x_scale, false);
        bind_tensor(e, a, &p.a, false);
        bind_tensor(e, b, &p.b, false);
        bind_tensor(e, adapterIds, &p.ids, false);
        bind_tensor(e, scaling, &p.scaling, false);
        bind_rows(e, out, &p.out, &p.ld_out, true);
        p.rows = rows; p.k = k; p.n = n; p.adapters = adapters; p.rank = rank;
        p.dtype = (int)base->dtype;
        p.x_i8 = x->dtype == ACL_INT8;
        e->kind = aclOpExecutor::kAdapterAdd;
        e->plan.ws_bytes = adapter_workspace_bytes(p);
    }
    return ne.hand_out(workspaceSize, executor);
}

// The weight of a dense product: rows along n, or along k in the transposed view of a weight stored [n, k]; any other view is copied.
void bind_weight(aclOpExecutor *e, const aclTensor *w, QuantMatmulProblem *p)
{
    const int64_t k = w->dim(0), n = w->dim(1), sk = w->strides[0], sn = w->strides[1];
    const bool by_n = (n == 1 || sn == 1) && (k == 1 || sk >= n), by_k = (k == 1 || sk == 1) && (n == 1 || sn >= k);
    p->w_nk = !by_n && by_k;
    p->ld_w = p->w_nk ? (n > 1 ? sn : k) : by_n && k > 1 ? sk : n;
    bind_tensor(e, w, &p->w, false, by_n || by_k);
}

aclnnStatus matmul_phase1(const aclTensor *x, const aclTensor *weight, const aclTensor *scale, const aclTensor *perTokenScale,
                          const aclTensor *bias, aclTensor *y, uint64_t *workspaceSize, aclOpExecutor **executor)
{
    REQUIRE_NOT_NULL(workspaceSize); REQUIRE_NOT_NULL(executor);
    REQUIRE_NOT_NULL(x); REQUIRE_NOT_NULL(weight); REQUIRE_NOT_NULL(scale); REQUIRE_NOT_NULL(y);
    REQUIRE_RANK(x, 2); REQUIRE_RANK(weight, 2);
    const int64_t m = x->dim(0), k = x->dim(1), n = weight->dim(1);
    GMM_REQUIRE(x->dtype == ACL_INT8 && weight->dtype == ACL_INT8, ACLNN_ERR_PARAM_INVALID, "x and weight dtype must be int8.");
    GMM_REQUIRE(m >= 0 && m <= kMaxRows, ACLNN_ERR_PARAM_INVALID, "x must not have more than %lld rows.", (long long)kMaxRows);
    GMM_REQUIRE(k >= 1 && k <= kMaxAxis, ACLNN_ERR_PARAM_INVALID, "k must be in [1, %lld], but is %lld.", (long long)kMaxAxis, (long long)k);
    GMM_REQUIRE(n >= 1 && n <= kMaxChannels, ACLNN_ERR_PARAM_INVALID, "n must be in [1, %lld], but is %lld.", (long long)kMaxChannels, (long long)n);
    REQUIRE_SHAPE2(weight, k, n);
    REQUIRE_SHAPE1(scale, n);
    GMM_REQUIRE(is_float(scale->dtype), ACLNN_ERR_PARAM_INVALID, "scale dtype must be float32, float16 or bfloat16.");
    if (perTokenScale) {
        REQUIRE_SHAPE1(perTokenScale, m);
        GMM_REQUIRE(perTokenScale->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "perTokenScale dtype must be float32.");
    }
    if (bias) {
        REQUIRE_SHAPE1(bias, n);
        GMM_REQUIRE(is_float(bias->dtype), ACLNN_ERR_PARAM_INVALID, "bias dtype must be float32, float16 or bfloat16.");
    }
    REQUIRE_SHAPE2(y, m, n);
    GMM_REQUIRE(is_float(y->dtype), ACLNN_ERR_PARAM_INVALID, "y dtype must be float32, float16 or bfloat16.");
    REQUIRE_USABLE(x, weight, scale, perTokenScale, bias, y);

    NewExecutor ne("gmmB200QuantMatmul");
    aclOpExecutor *e = ne.e;
    GMM_REQUIRE(e != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "cannot create executor.");
    if (m > 0) {
        QuantMatmulProblem &p = e->matmul;
        bind_rows(e, x, &p.x, &p.ld_x, false);
        bind_weight(e, weight, &p);
        bind_tensor(e, scale, &p.scale, false);
        bind_tensor(e, perTokenScale, &p.token_scale, false);
        bind_tensor(e, bias, &p.bias, false);
        bind_rows(e, y, &p.y, &p.ld_y, true);
        p.scale_dtype = (int)scale->dtype; p.bias_dtype = bias ? (int)bias->dtype : kNone; p.y_dtype = (int)y->dtype;
        p.m = m; p.k = k; p.n = n;
        e->kind = aclOpExecutor::kQuantMatmul;
        e->plan.ws_bytes = quant_matmul_workspace_bytes(p);
    }
    return ne.hand_out(workspaceSize, executor);
}

aclnnStatus sandwich_phase1(const aclTensor *x, const aclTensor *residual, const aclTensor *gamma, const aclTensor *postGamma,
                            const aclTensor *gate, const aclTensor *smooth, int64_t gateAct, float residualScale, float blockScale, float eps,
                            float postEps, aclTensor *q, aclTensor *scale, aclTensor *residualOut, aclTensor *normedOut,
                            uint64_t *workspaceSize, aclOpExecutor **executor)
{
    REQUIRE_NOT_NULL(workspaceSize); REQUIRE_NOT_NULL(executor);
    REQUIRE_NOT_NULL(x); REQUIRE_NOT_NULL(residual);
    GMM_REQUIRE(q || residualOut || normedOut, ACLNN_ERR_PARAM_NULLPTR, "one of q, residualOut and normedOut is needed.");
    GMM_REQUIRE((q == nullptr) == (scale == nullptr), ACLNN_ERR_PARAM_NULLPTR, "q and scale come together.");
    GMM_REQUIRE(gamma || (!q && !normedOut), ACLNN_ERR_PARAM_NULLPTR, "q and normedOut need gamma.");
    REQUIRE_RANK(residual, 2);
    const int64_t rows = residual->dim(0), h = residual->dim(1);
    const aclDataType type = residual->dtype;
    GMM_REQUIRE(is_float(type), ACLNN_ERR_PARAM_INVALID, "residual dtype must be float32, float16 or bfloat16.");
    GMM_REQUIRE(h >= 1 && h <= kMaxAxis, ACLNN_ERR_PARAM_INVALID, "residual's rows must have 1 to %lld elements, but have %lld.", (long long)kMaxAxis, (long long)h);
    GMM_REQUIRE(rows >= 0 && rows <= kMaxRows, ACLNN_ERR_PARAM_INVALID, "residual must not have more than %lld rows.", (long long)kMaxRows);
    REQUIRE_SHAPE2(x, rows, h);
    GMM_REQUIRE(x->dtype == type || x->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "x dtype must be residual's or float32.");
    const aclDataType gamma_type = gamma ? gamma->dtype : postGamma ? postGamma->dtype : type;
    GMM_REQUIRE(gamma_type == type || gamma_type == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "gamma and postGamma dtype must be residual's or float32.");
    for (const aclTensor *t : {gamma, postGamma})
        GMM_REQUIRE(!t || (t->rank() == 1 && t->dim(0) == h && t->dtype == gamma_type), ACLNN_ERR_PARAM_INVALID,
                    "gamma and postGamma must have shape [%lld] and the same dtype.", (long long)h);
    if (smooth) {
        REQUIRE_SHAPE1(smooth, h);
        GMM_REQUIRE(smooth->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "smooth dtype must be float32.");
    }
    if (gate) {
        const bool shape = gate->rank() == 1 ? gate->dim(0) == h
                           : gate->rank() == 2 && (gate->dim(0) == rows || gate->dim(0) == 1) && (gate->dim(1) == h || gate->dim(1) == 1);
        GMM_REQUIRE(shape, ACLNN_ERR_PARAM_INVALID, "gate shape must be [%lld], or [%lld or 1, %lld or 1].", (long long)h, (long long)rows, (long long)h);
        GMM_REQUIRE(gate->dtype == type, ACLNN_ERR_PARAM_INVALID, "gate dtype must be residual's.");
    }
    GMM_REQUIRE(gateAct >= kGateNone && gateAct <= kGateTanh, ACLNN_ERR_PARAM_INVALID, "gateAct must be 0 (none), 1 (sigmoid) or 2 (tanh).");
    if (q) {
        REQUIRE_SHAPE2(q, rows, h);
        GMM_REQUIRE(q->dtype == ACL_INT8, ACLNN_ERR_PARAM_INVALID, "q dtype must be int8.");
        REQUIRE_SHAPE1(scale, rows);
        GMM_REQUIRE(scale->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "scale dtype must be float32.");
    }
    for (const aclTensor *t : {residualOut, normedOut})
        GMM_REQUIRE(!t || (t->rank() == 2 && t->dim(0) == rows && t->dim(1) == h && t->dtype == type), ACLNN_ERR_PARAM_INVALID,
                    "residualOut and normedOut must have residual's shape and dtype.");
    REQUIRE_USABLE(x, residual, gamma, postGamma, gate, smooth, q, scale, residualOut, normedOut);
    GMM_REQUIRE(eps > 0.0f && std::isfinite(eps) && postEps > 0.0f && std::isfinite(postEps), ACLNN_ERR_PARAM_INVALID, "eps and postEps must be positive and finite.");
    GMM_REQUIRE(std::isfinite(residualScale) && std::isfinite(blockScale), ACLNN_ERR_PARAM_INVALID, "residualScale and blockScale must be finite.");

    NewExecutor ne("gmmB200SandwichNormQuant");
    aclOpExecutor *e = ne.e;
    GMM_REQUIRE(e != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "cannot create executor.");
    if (rows > 0) {
        SandwichNormProblem &p = e->sandwich;
        bind_rows(e, x, &p.x, &p.ld_x, false);
        bind_rows(e, residual, &p.residual, &p.ld_residual, false);
        bind_tensor(e, gamma, &p.gamma, false);
        bind_tensor(e, postGamma, &p.post_gamma, false);
        if (gate) {
            const bool wide = gate->rank() == 1 || gate->dim(1) == h, tall = gate->rank() == 2 && gate->dim(0) == rows && rows > 1;
            p.gate_step = wide && h > 1 ? 1 : 0;
            if (gate->rank() == 2 && p.gate_step == 0) {   // a column: used where it is, however far its elements are apart
                p.ld_gate = tall ? gate->strides[0] : 0;
                bind_tensor(e, gate, &p.gate, false, true);
            } else if (gate->rank() == 2) {
                bind_rows(e, gate, &p.gate, &p.ld_gate, false);
                if (!tall) p.ld_gate = 0;
            } else {
                bind_tensor(e, gate, &p.gate, false);
            }
        }
        bind_tensor(e, smooth, &p.smooth, false);
        bind_rows(e, q, &p.q, &p.ld_q, true);
        bind_tensor(e, scale, &p.scale, true);
        bind_rows(e, residualOut, &p.residual_out, &p.ld_residual_out, true);
        bind_rows(e, normedOut, &p.normed_out, &p.ld_normed, true);
        p.rows = rows; p.h = h;
        p.dtype = (int)type; p.x_dtype = (int)x->dtype; p.gamma_dtype = (int)gamma_type;
        p.gate_act = (int)gateAct;
        p.residual_scale = residualScale; p.block_scale = blockScale; p.eps = eps; p.post_eps = postEps;
        e->kind = aclOpExecutor::kSandwichNorm;
        e->plan.ws_bytes = kSandwichNormWorkspace;
    }
    return ne.hand_out(workspaceSize, executor);
}

// What the balance loss and its gradient share.
aclnnStatus check_balance(const aclTensor *logits, const aclTensor *tokenMask, const aclTensor *cuSeqlens, int64_t scoring, const aclTensor *counts,
                          const aclTensor *weight, int64_t *sequences)
{
    REQUIRE_NOT_NULL(logits); REQUIRE_NOT_NULL(counts); REQUIRE_NOT_NULL(weight);
    REQUIRE_RANK(logits, 2);
    const int64_t rows = logits->dim(0), experts = logits->dim(1);
    GMM_REQUIRE(is_float(logits->dtype), ACLNN_ERR_PARAM_INVALID, "logits dtype must be float32, float16 or bfloat16.");
    GMM_REQUIRE(experts >= 1 && experts <= 1024, ACLNN_ERR_PARAM_INVALID, "logits must name 1 to 1024 experts, but name %lld.", (long long)experts);
    GMM_REQUIRE(rows >= 0 && rows <= kMaxRows, ACLNN_ERR_PARAM_INVALID, "logits must not have more than %lld rows.", (long long)kMaxRows);
    GMM_REQUIRE(scoring == kScoreSoftmax || scoring == kScoreSigmoid, ACLNN_ERR_PARAM_INVALID, "scoring must be 0 (softmax) or 1 (sigmoid).");
    if (tokenMask) {
        REQUIRE_SHAPE1(tokenMask, rows);
        GMM_REQUIRE(tokenMask->dtype == ACL_INT8 || tokenMask->dtype == ACL_BOOL, ACLNN_ERR_PARAM_INVALID, "tokenMask dtype must be int8 or bool.");
    }
    *sequences = 1;
    if (cuSeqlens) {
        REQUIRE_RANK(cuSeqlens, 1);
        GMM_REQUIRE(cuSeqlens->dtype == ACL_INT32, ACLNN_ERR_PARAM_INVALID, "cuSeqlens dtype must be int32.");
        *sequences = cuSeqlens->dim(0) - 1;
        GMM_REQUIRE(*sequences >= 1 && *sequences <= kMaxAxis, ACLNN_ERR_PARAM_INVALID, "cuSeqlens must name 1 to %lld sequences, but names %lld.",
                    (long long)kMaxAxis, (long long)*sequences);
        REQUIRE_SHAPE2(counts, *sequences, experts);
    } else {
        REQUIRE_SHAPE1(counts, experts);
    }
    GMM_REQUIRE(counts->dtype == ACL_INT64, ACLNN_ERR_PARAM_INVALID, "counts dtype must be int64.");
    REQUIRE_SHAPE1(weight, *sequences);
    GMM_REQUIRE(weight->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "weight dtype must be float32.");
    return ACLNN_SUCCESS;
}

void bind_balance(aclOpExecutor *e, const aclTensor *logits, const aclTensor *tokenMask, const aclTensor *cuSeqlens, int64_t scoring, int64_t sequences)
{
    BalanceProblem &p = e->balance;
    bind_rows(e, logits, &p.logits, &p.ld, false);
    p.dtype = (int)logits->dtype;
    bind_tensor(e, tokenMask, &p.token_mask, false);
    bind_tensor(e, cuSeqlens, &p.cu_seqlens, false);
    p.rows = logits->dim(0); p.experts = (int)logits->dim(1); p.sequences = sequences;
    p.scoring = (int)scoring;
}

aclnnStatus balance_phase1(const aclTensor *logits, const aclTensor *ids, const aclTensor *tokenMask, const aclTensor *cuSeqlens, int64_t scoring,
                           float coefficient, aclTensor *loss, aclTensor *counts, aclTensor *weight, uint64_t *workspaceSize,
                           aclOpExecutor **executor)
{
    REQUIRE_NOT_NULL(workspaceSize); REQUIRE_NOT_NULL(executor);
    REQUIRE_NOT_NULL(ids); REQUIRE_NOT_NULL(loss);
    int64_t sequences = 1;
    const aclnnStatus rc = check_balance(logits, tokenMask, cuSeqlens, scoring, counts, weight, &sequences);
    if (rc != ACLNN_SUCCESS) return rc;
    REQUIRE_RANK(ids, 2);
    GMM_REQUIRE(ids->dim(0) == logits->dim(0) && ids->dim(1) >= 1 && ids->dim(1) <= 1024, ACLNN_ERR_PARAM_INVALID,
                "ids shape must be [%lld, 1 to 1024].", (long long)logits->dim(0));
    GMM_REQUIRE(ids->dtype == ACL_INT32 || ids->dtype == ACL_INT64, ACLNN_ERR_PARAM_INVALID, "ids dtype must be int32 or int64.");
    GMM_REQUIRE(loss->numel() == 1 && loss->dtype == ACL_FLOAT, ACLNN_ERR_PARAM_INVALID, "loss must be one float32 element.");
    GMM_REQUIRE(std::isfinite(coefficient), ACLNN_ERR_PARAM_INVALID, "coefficient must be finite.");
    REQUIRE_USABLE(logits, ids, tokenMask, cuSeqlens, loss, counts, weight);

    NewExecutor ne("gmmB200ExpertBalance");
    aclOpExecutor *e = ne.e;
    GMM_REQUIRE(e != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "cannot create executor.");
    BalanceProblem &p = e->balance;
    bind_balance(e, logits, tokenMask, cuSeqlens, scoring, sequences);
    bind_tensor(e, ids, &p.ids, false);
    bind_tensor(e, loss, &p.loss, true);
    bind_tensor(e, counts, &p.counts, true);
    bind_tensor(e, weight, &p.weight, true);
    p.ids_i64 = ids->dtype == ACL_INT64;
    p.top_k = (int)ids->dim(1);
    p.coefficient = coefficient;
    e->kind = aclOpExecutor::kBalance;   // without rows, too: the loss is 0 then
    e->plan.ws_bytes = balance_workspace_bytes(p);
    return ne.hand_out(workspaceSize, executor);
}

aclnnStatus balance_grad_phase1(const aclTensor *logits, const aclTensor *counts, const aclTensor *weight, const aclTensor *tokenMask,
                                const aclTensor *cuSeqlens, const aclTensor *gradLoss, int64_t scoring, aclTensor *grad, uint64_t *workspaceSize,
                                aclOpExecutor **executor)
{
    REQUIRE_NOT_NULL(workspaceSize); REQUIRE_NOT_NULL(executor);
    REQUIRE_NOT_NULL(grad);
    int64_t sequences = 1;
    const aclnnStatus rc = check_balance(logits, tokenMask, cuSeqlens, scoring, counts, weight, &sequences);
    if (rc != ACLNN_SUCCESS) return rc;
    GMM_REQUIRE(!gradLoss || (gradLoss->numel() == 1 && gradLoss->dtype == ACL_FLOAT), ACLNN_ERR_PARAM_INVALID, "gradLoss must be one float32 element.");
    REQUIRE_SHAPE2(grad, logits->dim(0), logits->dim(1));
    GMM_REQUIRE(grad->dtype == logits->dtype, ACLNN_ERR_PARAM_INVALID, "grad dtype must be logits'.");
    REQUIRE_USABLE(logits, counts, weight, tokenMask, cuSeqlens, gradLoss, grad);

    NewExecutor ne("gmmB200ExpertBalanceGrad");
    aclOpExecutor *e = ne.e;
    GMM_REQUIRE(e != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "cannot create executor.");
    if (logits->dim(0) > 0) {
        BalanceProblem &p = e->balance;
        bind_balance(e, logits, tokenMask, cuSeqlens, scoring, sequences);
        bind_tensor(e, counts, &p.counts, false);
        bind_tensor(e, weight, &p.weight, false);
        bind_tensor(e, gradLoss, &p.grad_loss, false);
        bind_rows(e, grad, &p.grad, &p.ld_grad, true);
        e->kind = aclOpExecutor::kBalanceGrad;
    }
    return ne.hand_out(workspaceSize, executor);
}

// A first phase whose allocations may fail.
template <typename Fn>
aclnnStatus guarded(const char *name, Fn fn)
{
    try {
        clear_error();
        PhaseRange phase_range(name, 1);
        return fn();
    } catch (const std::exception &ex) {
        return fail(ACLNN_ERR_INNER_CREATE_EXECUTOR, "%s: %s", name, ex.what());
    }
}

}  // namespace
}  // namespace gmm

using namespace gmm;

extern "C" {

aclnnStatus gmmB200AddRmsNormQuantGetWorkspaceSize(const aclTensor *x, const aclTensor *residualOptional, const aclTensor *gamma,
                                                   const aclTensor *smoothOptional, float eps, aclTensor *q, aclTensor *scale,
                                                   aclTensor *residualOutOptional, aclTensor *normedOutOptional, uint64_t *workspaceSize,
                                                   aclOpExecutor **executor)
{
    return guarded("gmmB200AddRmsNormQuant", [&] {
        return norm_phase1(x, residualOptional, gamma, smoothOptional, eps, q, scale, residualOutOptional, normedOutOptional, workspaceSize, executor);
    });
}

aclnnStatus gmmB200AddRmsNormQuant(void *workspace, uint64_t workspaceSize, aclOpExecutor *executor, aclrtStream stream)
{
    return run_executor("gmmB200AddRmsNormQuant", workspace, workspaceSize, executor, stream);
}

aclnnStatus gmmB200RouteTopKGetWorkspaceSize(const aclTensor *logits, const aclTensor *biasOptional, const aclTensor *tokenMaskOptional,
                                             int64_t scoring, int64_t nGroup, int64_t topkGroup, int64_t groupScore, bool renormalize,
                                             float scale, aclTensor *weights, aclTensor *ids, uint64_t *workspaceSize, aclOpExecutor **executor)
{
    return guarded("gmmB200RouteTopK", [&] {
        return route_phase1(logits, biasOptional, tokenMaskOptional, scoring, nGroup, topkGroup, groupScore, renormalize, scale, weights, ids,
                            workspaceSize, executor);
    });
}

aclnnStatus gmmB200RouteTopK(void *workspace, uint64_t workspaceSize, aclOpExecutor *executor, aclrtStream stream)
{
    return run_executor("gmmB200RouteTopK", workspace, workspaceSize, executor, stream);
}

aclnnStatus gmmB200AdapterAddGetWorkspaceSize(const aclTensor *base, const aclTensor *x, const aclTensor *xScaleOptional, const aclTensor *a,
                                              const aclTensor *b, const aclTensor *adapterIds, const aclTensor *scalingOptional,
                                              aclTensor *out, uint64_t *workspaceSize, aclOpExecutor **executor)
{
    return guarded("gmmB200AdapterAdd", [&] {
        return adapter_phase1(base, x, xScaleOptional, a, b, adapterIds, scalingOptional, out, workspaceSize, executor);
    });
}

aclnnStatus gmmB200AdapterAdd(void *workspace, uint64_t workspaceSize, aclOpExecutor *executor, aclrtStream stream)
{
    return run_executor("gmmB200AdapterAdd", workspace, workspaceSize, executor, stream);
}

aclnnStatus gmmB200QuantMatmulGetWorkspaceSize(const aclTensor *x, const aclTensor *weight, const aclTensor *scale,
                                               const aclTensor *perTokenScaleOptional, const aclTensor *biasOptional, aclTensor *y,
                                               uint64_t *workspaceSize, aclOpExecutor **executor)
{
    return guarded("gmmB200QuantMatmul", [&] { return matmul_phase1(x, weight, scale, perTokenScaleOptional, biasOptional, y, workspaceSize, executor); });
}

aclnnStatus gmmB200QuantMatmul(void *workspace, uint64_t workspaceSize, aclOpExecutor *executor, aclrtStream stream)
{
    return run_executor("gmmB200QuantMatmul", workspace, workspaceSize, executor, stream);
}

aclnnStatus gmmB200SandwichNormQuantGetWorkspaceSize(const aclTensor *x, const aclTensor *residual, const aclTensor *gammaOptional,
                                                     const aclTensor *postGammaOptional, const aclTensor *gateOptional,
                                                     const aclTensor *smoothOptional, int64_t gateAct, float residualScale, float blockScale,
                                                     float eps, float postEps, aclTensor *qOptional, aclTensor *scaleOptional,
                                                     aclTensor *residualOutOptional, aclTensor *normedOutOptional, uint64_t *workspaceSize,
                                                     aclOpExecutor **executor)
{
    return guarded("gmmB200SandwichNormQuant", [&] {
        return sandwich_phase1(x, residual, gammaOptional, postGammaOptional, gateOptional, smoothOptional, gateAct, residualScale, blockScale, eps,
                               postEps, qOptional, scaleOptional, residualOutOptional, normedOutOptional, workspaceSize, executor);
    });
}

aclnnStatus gmmB200SandwichNormQuant(void *workspace, uint64_t workspaceSize, aclOpExecutor *executor, aclrtStream stream)
{
    return run_executor("gmmB200SandwichNormQuant", workspace, workspaceSize, executor, stream);
}

aclnnStatus gmmB200ExpertBalanceGetWorkspaceSize(const aclTensor *logits, const aclTensor *ids, const aclTensor *tokenMaskOptional,
                                                 const aclTensor *cuSeqlensOptional, int64_t scoring, float coefficient, aclTensor *loss,
                                                 aclTensor *counts, aclTensor *weight, uint64_t *workspaceSize, aclOpExecutor **executor)
{
    return guarded("gmmB200ExpertBalance", [&] {
        return balance_phase1(logits, ids, tokenMaskOptional, cuSeqlensOptional, scoring, coefficient, loss, counts, weight, workspaceSize, executor);
    });
}

aclnnStatus gmmB200ExpertBalance(void *workspace, uint64_t workspaceSize, aclOpExecutor *executor, aclrtStream stream)
{
    return run_executor("gmmB200ExpertBalance", workspace, workspaceSize, executor, stream);
}

aclnnStatus gmmB200ExpertBalanceGradGetWorkspaceSize(const aclTensor *logits, const aclTensor *counts, const aclTensor *weight,
                                                     const aclTensor *tokenMaskOptional, const aclTensor *cuSeqlensOptional,
                                                     const aclTensor *gradLossOptional, int64_t scoring, aclTensor *grad, uint64_t *workspaceSize,
                                                     aclOpExecutor **executor)
{
    return guarded("gmmB200ExpertBalanceGrad", [&] {
        return balance_grad_phase1(logits, counts, weight, tokenMaskOptional, cuSeqlensOptional, gradLossOptional, scoring, grad, workspaceSize, executor);
    });
}

aclnnStatus gmmB200ExpertBalanceGrad(void *workspace, uint64_t workspaceSize, aclOpExecutor *executor, aclrtStream stream)
{
    return run_executor("gmmB200ExpertBalanceGrad", workspace, workspaceSize, executor, stream);
}

}  // extern "C"
