// What the entry points of include/tenmo_hip_transformer.h share: errors, the device they launch on, the caller's
// workspace, views as the kernels take them, and the reductions across a wavefront and a workgroup.
#ifndef TENMO_KERNELS_ENTRY_HPP
#define TENMO_KERNELS_ENTRY_HPP
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/tenmo_hip_transformer.h"
#include "../csrc/library_state.hpp"

namespace tenmo {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at a 4-byte boundary: global memory takes such an access as one instruction
typedef f32x4 f32x4_u __attribute__((aligned(4)));

__attribute__((format(printf, 2, 3))) inline int refuse(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return library_error(code, buf);
}

// The library's stream, on the library's device: a caller whose current device is another one keeps it.
class Call {
public:
    explicit Call(const char* who) : who_(who) {}
    ~Call() {
        if (previous_ >= 0) (void)hipSetDevice(previous_);
    }
    int begin() {
        if (int rc = library_state(&state)) return rc;
        int current = -1;
        if (int rc = check(hipGetDevice(&current), "hipGetDevice")) return rc;
        if (current != state.device) {
            if (int rc = check(hipSetDevice(state.device), "hipSetDevice")) return rc;
            previous_ = current;
        }
        return 0;
    }
    int finish(int32_t sync) {
        if (int rc = check(hipGetLastError(), "kernel launch")) return rc;
        return sync ? check(hipStreamSynchronize(state.stream), "hipStreamSynchronize") : 0;
    }
    LibraryState state{};

private:
    int check(hipError_t e, const char* what) {
        return e == hipSuccess ? 0 : refuse(TENMO_ERR_HIP, "%s: %s failed: %s", who_, what, hipGetErrorString(e));
    }
    const char* who_;
    int previous_ = -1;
};

// Pieces of the caller's workspace, 256-byte aligned.  With no base it only adds the sizes up.
class Workspace {
public:
    Workspace(void* base, int64_t bytes) : base_((char*)base), bytes_(bytes) {}
    template <class T>
    T* take(int64_t count) {
        const int64_t at = used_;
        used_ += (count * (int64_t)sizeof(T) + 255) / 256 * 256;
        return base_ ? (T*)(base_ + at) : nullptr;
    }
    int64_t used() const { return used_; }
    int check(const char* who) const {
        if (used_ && (!base_ || used_ > bytes_))
            return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, %lld needed", who, base_ ? (long long)bytes_ : 0LL, (long long)used_);
        if ((uintptr_t)base_ % 256) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: workspace is not aligned to 256 bytes", who);
        return 0;
    }

private:
    char* base_;
    int64_t bytes_, used_ = 0;
};

inline int check_operand(const tenmo_view* v, int min_rank, int max_rank, const char* who, const char* what) {
    if (!v) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: null %s", who, what);
    if (v->rank < min_rank || v->rank > max_rank)
        return refuse(TENMO_ERR_INVALID_SHAPE, "%s: %s has rank %d, needs %d to %d", who, what, v->rank, min_rank, max_rank);
    int64_t n = 1;
    for (int d = 0; d < v->rank; ++d) {
        if (v->shape[d] < 0) return refuse(TENMO_ERR_INVALID_SHAPE, "%s: %s has a negative dimension", who, what);
        n = v->shape[d] && n > INT64_MAX / v->shape[d] ? INT64_MAX : n * v->shape[d];
    }
    if (n == INT64_MAX) return refuse(TENMO_ERR_INVALID_SHAPE, "%s: %s has too many elements", who, what);
    if (n > 0 && !v->data) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: %s has no data", who, what);
    return 0;
}

inline int64_t elements(const tenmo_view* v) {
    int64_t n = 1;
    for (int d = 0; d < v->rank; ++d) n *= v->shape[d];
    return n;
}

// ---- reductions ---------------------------------------------------------------------------------------------------------
// Between lanes through the vector unit's own lane moves (no LDS): within quads, halves of 16, 16, then rows of 16 exchanged.  Every lane ends with the same
// bits: each step adds the same two values in either order.

template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// f(this lane's group of L, the neighbouring one's) for L = 1, 2, 4 .. 64 / 2
template <int L, class F>
__device__ __forceinline__ float lanes_reduce(float v, F f) {
    if (L >= 2) v = f(v, lane_move<0xB1>(v));   // quad_perm 1 0 3 2
    if (L >= 4) v = f(v, lane_move<0x4E>(v));   // quad_perm 2 3 0 1
    if (L >= 8) v = f(v, lane_move<0x141>(v));  // row_half_mirror
    if (L >= 16) v = f(v, lane_move<0x140>(v)); // row_mirror
    if (L >= 32) {
        const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    if (L >= 64) {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    return v;
}
// over each group of L lanes
template <int L>
__device__ __forceinline__ float lanes_sum(float v) { return lanes_reduce<L>(v, [](float a, float b) { return a + b; }); }
template <int L>
__device__ __forceinline__ float lanes_max(float v) { return lanes_reduce<L>(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float wave_sum(float v) { return lanes_sum<64>(v); }
__device__ __forceinline__ float wave_max(float v) { return lanes_max<64>(v); }
// of this lane and the one 32 further
__device__ __forceinline__ float halves_max(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// The sum over W wavefronts of a workgroup, in every thread, the same bits in all of them.  `slots` holds W floats; calls that
// follow each other alternate between two sets of slots.
template <int W>
__device__ __forceinline__ float group_sum(float v, float* slots) {
    v = wave_sum(v);
    if (W == 1) return v;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) slots[wave] = v;
    __syncthreads();
    float s = slots[0];
#pragma unroll
    for (int i = 1; i < W; ++i) s += slots[i];
    return s;
}

} // namespace tenmo
#endif
