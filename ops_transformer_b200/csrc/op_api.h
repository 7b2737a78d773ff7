// What the first phases of all operators share: checks, executors, the binding of tensors, profiler ranges.
#pragma once
#include <nvtx3/nvToolsExt.h>

#include <cstdio>
#include <cstdlib>
#include <new>

#include "acl_shim.h"

#define GMM_REQUIRE(cond, code, ...)                   \
    do {                                               \
        if (!(cond)) return fail((code), __VA_ARGS__); \
    } while (0)

namespace gmm {

void register_executor(aclOpExecutor *e);
bool claim_executor(aclOpExecutor *e);
bool executor_is_live(aclOpExecutor *e);

inline bool is_private_format(aclFormat f) { return f == ACL_FORMAT_FRACTAL_NZ || f == ACL_FORMAT_FRACTAL_Z || f == ACL_FORMAT_NC1HWC0; }

inline aclOpExecutor *new_executor(const char *name)
{
    aclOpExecutor *e = new (std::nothrow) aclOpExecutor();
    if (e) e->op_name = name;
    return e;
}

// Address the operator will use for tensor `t`: the tensor's own memory when it is contiguous; otherwise a contiguous
// copy in the workspace tail, filled before the launch (and, for an output, copied back afterwards).  The address of a
// copy is only known in the second phase: until then `*field` holds an aligned stand-in.
template <typename P>
void bind_tensor(aclOpExecutor *e, const aclTensor *t, P *field, bool is_output, bool contiguous_enough = false)
{
    if (!t) { *field = nullptr; return; }
    if (t->contiguous() || contiguous_enough) { *field = (P)tensor_ptr(t); return; }
    StagedView v;
    v.dims.assign(t->view_dims.begin(), t->view_dims.end());
    v.strides.assign(t->strides.begin(), t->strides.end());
    v.elem = (int)dtype_size(t->dtype);
    v.data = tensor_ptr(t);
    v.ws_off = e->staged_bytes;
    v.is_output = is_output;
    v.field = (void **)field;  // the field is a pointer of some type; only its value is replaced
    e->staged_bytes += ((size_t)t->numel() * v.elem + 255) / 256 * 256;
    e->staged.push_back(v);
    *field = (P)(uintptr_t)4096;
}

// The same for rows of a matrix: a view whose rows are dense is used where it is, with its row stride in *ld (elements).  Rows of
// an output must not share memory.
template <typename P>
void bind_rows(aclOpExecutor *e, const aclTensor *t, P *field, int64_t *ld, bool is_output)
{
    if (!t) { *field = nullptr; *ld = 0; return; }
    const int64_t rows = t->dim(0), cols = t->dim(1);
    const bool dense = (cols == 1 || t->strides[1] == 1) && (rows == 1 || t->strides[0] >= (is_output ? cols : 0));
    *ld = dense && rows > 1 ? t->strides[0] : cols;
    bind_tensor(e, t, field, is_output, dense);
}

// Env-gated profiler ranges around both phases of every entry point (GMM_B200_NVTX=1), the counterpart of the
// reference's L2_DFX_PHASE_1 / L2_DFX_PHASE_2 (gmm/grouped_matmul/op_host/op_api/aclnn_grouped_matmul.cpp:2005, 2151).
// NVTX is header only and does nothing unless a tool is attached.
inline bool nvtx_enabled()
{
    static const bool on = [] {
        const char *e = std::getenv("GMM_B200_NVTX");
        return e && e[0] && e[0] != '0';
    }();
    return on;
}
struct PhaseRange {
    bool on;
    PhaseRange(const char *op, int phase) : on(nvtx_enabled())
    {
        if (!on) return;
        char name[160];
        std::snprintf(name, sizeof(name), "%s phase %d", op, phase);
        nvtxRangePushA(name);
    }
    ~PhaseRange()
    {
        if (on) nvtxRangePop();
    }
};

inline aclnnStatus finish_phase1(aclOpExecutor *e, uint64_t *workspaceSize, aclOpExecutor **executor)
{
    // every kind stores its size in plan.ws_bytes
    *workspaceSize = e->kind == aclOpExecutor::kNoop ? 0 : e->plan.ws_bytes + e->staged_bytes;
    register_executor(e);
    *executor = e;
    return ACLNN_SUCCESS;
}

}  // namespace gmm
