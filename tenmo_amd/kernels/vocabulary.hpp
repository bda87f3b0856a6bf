// What the kernels of the vocabulary loss share: the call, its targets and the factor of each row's gradient.
#ifndef TENMO_KERNELS_VOCABULARY_HPP
#define TENMO_KERNELS_VOCABULARY_HPP
#include "entry.hpp"

namespace tenmo {

struct VocabArgs {
    int64_t M, V, D;
    const float* bias;
    const void* target;
    int is64;
    int64_t ignore;
    float ls;
};

__device__ __forceinline__ int64_t target_of(const VocabArgs& a, int64_t m) {
    return a.is64 ? ((const int64_t*)a.target)[m] : (int64_t)((const int32_t*)a.target)[m];
}

struct Upstream { // the gradient of the loss: of each row, or of the reduced one
    const float* p;
    int reduction;
    const int32_t* valid_count;
};
// the factor of row m of the gradient; 0 where the target is ignore_index
__device__ __forceinline__ float row_factor(const VocabArgs& a, const Upstream& u, int64_t m) {
    if (target_of(a, m) == a.ignore) return 0.f;
    const float s = u.p[u.reduction == 0 ? m : 0];
    return u.reduction == 2 ? s / (float)(*u.valid_count > 1 ? *u.valid_count : 1) : s;
}

struct Operand2 { // element (r, c) of a view of rank 2
    const float* p;
    int64_t r, c;
};

// ---- few tokens, or a small W: vocabulary_few.hip ----
bool few_for_forward(int64_t tokens, int64_t dim, int64_t words);
bool few_for_backward(int64_t tokens, int64_t dim, int64_t words);
struct FewPlan {
    float2* part;       // [tiles][tokens], forward
    float *part_x, *target_logit;
    int64_t tiles;
    float* g;           // [tokens][words], backward
    float* part_h;      // [runs][tokens][dim]
    int64_t run, runs;  // words of a run
};
void few_plan_forward(Workspace& ws, FewPlan& p, const VocabArgs& v);
void few_plan_backward(Workspace& ws, FewPlan& p, const VocabArgs& v);
void few_forward(const FewPlan& p, const VocabArgs& v, const Operand2& h, const Operand2& w, hipStream_t stream);
// G into p.g, the runs of G W^T into p.part_h if `want_h`, (scale H)^T G into grad_w and the sums of scale G into grad_bias if they are not NULL
void few_backward(const FewPlan& p, const VocabArgs& v, const Operand2& h, const Operand2& w, const float* lse, const Upstream& up, bool want_h,
                  float* grad_w, int64_t gw_d, int64_t gw_v, float* grad_bias, int accumulate, hipStream_t stream);

} // namespace tenmo
#endif
