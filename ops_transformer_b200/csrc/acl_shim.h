// Concrete definitions of the opaque aclnn handle types (internal).
#pragma once
#include <cstdarg>
#include <cstdint>
#include <string>
#include <vector>

#include "aclnn/aclnn_base.h"
#include "gmm_common.h"

// Sizes of at most 8 dimensions, in place: a call describes up to ten tensors by three lists each, which as vectors were thirty
// allocations.
class Dims {
public:
    size_t size() const { return n_; }
    int64_t operator[](size_t i) const { return v_[i]; }
    int64_t &operator[](size_t i) { return v_[i]; }
    const int64_t *begin() const { return v_; }
    const int64_t *end() const { return v_ + n_; }
    int64_t *begin() { return v_; }
    int64_t *end() { return v_ + n_; }
    void resize(size_t n) { n_ = n; }   // n <= 8; the values are set next
    void assign(size_t n, int64_t v)
    {
        n_ = n;
        for (int64_t &d : *this) d = v;
    }
    void assign(const int64_t *from, const int64_t *to)
    {
        n_ = 0;
        while (from != to) v_[n_++] = *from++;
    }

private:
    size_t n_ = 0;
    int64_t v_[8];
};

struct aclTensor {
    Dims view_dims;
    Dims strides;                   // elements
    int64_t offset = 0;             // elements
    aclDataType dtype = ACL_DT_UNDEFINED;
    aclFormat format = ACL_FORMAT_ND;
    Dims storage_dims;
    void *data = nullptr;

    size_t rank() const { return view_dims.size(); }
    int64_t dim(size_t i) const { return view_dims[i]; }
    int64_t numel() const
    {
        int64_t n = 1;
        for (int64_t d : view_dims) n *= d;
        return n;
    }
    bool empty() const { return numel() == 0; }
    bool contiguous() const
    {
        int64_t expect = 1;
        for (size_t i = view_dims.size(); i-- > 0;) {
            if (view_dims[i] != 1 && strides[i] != expect) return false;
            expect *= view_dims[i];
        }
        return true;
    }
};

struct aclTensorList {
    std::vector<const aclTensor *> items;
};

struct aclIntArray {
    std::vector<int64_t> values;
};

struct aclOpExecutor {
    enum Kind { kNoop = 0, kGmm = 1, kInitRouting = 2, kNormQuant = 3, kRouteTopK = 4, kAdapterAdd = 5 } kind = kNoop;
    uint32_t magic = 0xac10e8ecu;
    bool consumed = false;
    const char *op_name = "";
    gmm::Problem problem;
    gmm::Plan plan;
    gmm::InitRoutingProblem routing;
    gmm::NormQuantProblem norm;
    gmm::RouteTopKProblem route;
    gmm::AdapterProblem adapter;
    std::vector<gmm::StagedView> staged;   // non-contiguous views with a contiguous copy in the workspace tail
    size_t staged_bytes = 0;
};

namespace gmm {

size_t dtype_size(aclDataType t);
// Stores a printf-style message as the calling thread's most recent error and returns `code`.
aclnnStatus fail(aclnnStatus code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();
// Element address of a tensor view's first element.
inline void *tensor_ptr(const aclTensor *t)
{
    return static_cast<char *>(t->data) + (size_t)t->offset * dtype_size(t->dtype);
}
aclnnStatus run_executor(const char *op_name, void *workspace, uint64_t workspace_size, aclOpExecutor *executor,
                         aclrtStream stream);

}  // namespace gmm
