// Layer norm over the last axis, forward and backward (include/tenmo_hip_transformer.h).
//
//   xhat = (x - mean) * rstd,  y = xhat * w + b
//   g = dy * w:  dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),  dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// Bound: HBM, 8 bytes an element forward (x read, y written), 12 backward (x and dy read, dx written).  A row is held in registers
// between its two passes (the mean, then the squares around it: no cancellation), so that each element is read once.
//   * up to 1024 columns: a wavefront per row, no barrier; up to 8192: a workgroup of 4 wavefronts per row; wider rows, and rows without
//     unit stride, are read again for each pass (from the caches) by norm_*_any_kernel.
//   * loads and stores are 16 bytes whatever the row's alignment (global memory needs 4): rows of odd length cost split cache lines,
//     not instructions.
//   * backward: each wavefront (or workgroup) takes every G-th row and keeps the sums of its columns for dw and db in registers; a row of partial sums a workgroup
//     goes to the workspace, and a second launch adds them in a fixed order.  For few rows workgroups of columns in the one launch take their place, unless grad_X is
//     written where they read.
#include "entry.hpp"

#include <algorithm>

namespace tenmo {
namespace {

struct NormRows {
    const float* x;
    int64_t rows, n;
    int64_t col_stride;
    int rank; // leading axes
    int64_t shape[TENMO_MAX_RANK], stride[TENMO_MAX_RANK];
};

__device__ __forceinline__ const float* norm_row(const NormRows& a, int64_t row) {
    int64_t off = 0;
    for (int d = a.rank - 1; d > 0; --d) {
        const int64_t q = row / a.shape[d];
        off += (row - q * a.shape[d]) * a.stride[d];
        row = q;
    }
    return a.x + off + (a.rank > 0 ? row * a.stride[0] : 0);
}

// element e (of 4) of this thread's k-th group is column 4 * (thread + threads * k) + e
template <int T, int V4>
__device__ __forceinline__ void load_row(f32x4 (&v)[V4], const float* __restrict p, int n, int t) {
#pragma unroll
    for (int k = 0; k < V4; ++k) {
        const int c = 4 * (t + T * k);
        if (c + 3 < n) v[k] = *(const f32x4_u*)(p + c);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][e] = c + e < n ? p[c + e] : 0.f;
    }
}

template <int T, int V4>
__device__ __forceinline__ void store_row(float* __restrict p, const f32x4 (&v)[V4], int n, int t) {
#pragma unroll
    for (int k = 0; k < V4; ++k) {
        const int c = 4 * (t + T * k);
        if (c + 3 < n) *(f32x4_u*)(p + c) = v[k];
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < n) p[c + e] = v[k][e];
    }
}

struct NormForward {
    NormRows in;
    const float *weight, *bias;
    float eps;
    float *out, *mean, *rstd;
};

// W wavefronts a row, V4 groups of 4 columns a thread; the workgroup is 256 threads.
template <int W, int V4>
__global__ __launch_bounds__(256) void norm_forward_kernel(const NormForward a) {
    constexpr int T = W * 64;
    __shared__ float slots[2][4];
    const int t = threadIdx.x % T, n = (int)a.in.n;
    for (int64_t row = (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T; row < a.in.rows; row += (int64_t)gridDim.x * (256 / T)) {
        f32x4 x[V4];
        load_row<T, V4>(x, norm_row(a.in, row), n, t);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < V4; ++k) s += (x[k][0] + x[k][1]) + (x[k][2] + x[k][3]);
        const float mean = group_sum<W>(s, slots[0]) / (float)n;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < V4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = 4 * (t + T * k) + e < n ? x[k][e] - mean : 0.f;
                x[k][e] = d;
                s += d * d;
            }
        const float rstd = 1.f / sqrtf(group_sum<W>(s, slots[1]) / (float)n + a.eps);
        f32x4 w[V4];
        if (a.weight) {
            load_row<T, V4>(w, a.weight, n, t);
#pragma unroll
            for (int k = 0; k < V4; ++k) x[k] = x[k] * rstd * w[k];
        } else {
#pragma unroll
            for (int k = 0; k < V4; ++k) x[k] = x[k] * rstd;
        }
        if (a.bias) {
            load_row<T, V4>(w, a.bias, n, t);
#pragma unroll
            for (int k = 0; k < V4; ++k) x[k] += w[k];
        }
        store_row<T, V4>(a.out + row * a.in.n, x, n, t);
        if (t == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

__global__ __launch_bounds__(256) void norm_forward_any_kernel(const NormForward a) {
    __shared__ float slots[2][4];
    const int64_t n = a.in.n, cs = a.in.col_stride;
    for (int64_t row = blockIdx.x; row < a.in.rows; row += gridDim.x) {
        const float* __restrict p = norm_row(a.in, row);
        float s = 0.f;
        for (int64_t c = threadIdx.x; c < n; c += 256) s += p[c * cs];
        const float mean = group_sum<4>(s, slots[0]) / (float)n;
        s = 0.f;
        for (int64_t c = threadIdx.x; c < n; c += 256) {
            const float d = p[c * cs] - mean;
            s += d * d;
        }
        const float rstd = 1.f / sqrtf(group_sum<4>(s, slots[1]) / (float)n + a.eps);
        for (int64_t c = threadIdx.x; c < n; c += 256) {
            const float y = (p[c * cs] - mean) * rstd * (a.weight ? a.weight[c] : 1.f);
            a.out[row * n + c] = a.bias ? y + a.bias[c] : y;
        }
        if (threadIdx.x == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

struct NormBackward {
    NormRows in;
    const float *weight, *mean, *rstd, *dy;
    float *grad_x, *grad_weight, *grad_bias;
    float* partial; // [parts][2][n]: sums of dy * xhat and of dy; NULL when neither is wanted, or the launch has workgroups for them
    int64_t parts;
    int accumulate;
    int64_t row_groups; // workgroups of rows; those behind them take 16 columns of dw and db each
};

// dw and db of 16 columns over all rows: 16 rows at a time, eight of each thread's in flight, their sums added in order
__device__ __forceinline__ void norm_columns(const NormBackward& a, int64_t group) {
    __shared__ float sums[2][16][16];
    const int64_t n = a.in.n, column = group * 16 + (threadIdx.x & 15), c = column < n ? column : n - 1;
    const int slot = threadIdx.x >> 4;
    float sw = 0.f, sb = 0.f;
#pragma unroll 8
    for (int64_t row = slot; row < a.in.rows; row += 16) {
        const float dy = a.dy[row * n + c];
        sw += dy * ((norm_row(a.in, row)[c * a.in.col_stride] - a.mean[row]) * a.rstd[row]);
        sb += dy;
    }
    sums[0][slot][threadIdx.x & 15] = sw;
    sums[1][slot][threadIdx.x & 15] = sb;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const int which = threadIdx.x >> 4, i = threadIdx.x & 15;
    float* out = which ? a.grad_bias : a.grad_weight;
    if (!out || column >= n) return;
    float s = sums[which][0][i];
#pragma unroll
    for (int k = 1; k < 16; ++k) s += sums[which][k][i];
    out[c] = a.accumulate ? out[c] + s : s;
}

// A row's x and dy are read while the row before it is worked on, where the registers allow.
template <int W, int V4>
__global__ __launch_bounds__(256) void norm_backward_kernel(const NormBackward a) {
    if (blockIdx.x >= a.row_groups) return norm_columns(a, blockIdx.x - a.row_groups);
    constexpr int T = W * 64, R = 256 / T; // rows a workgroup works on at a time
    constexpr bool AHEAD = V4 <= 4;
    __shared__ float slots[2][2][4];
    const int t = threadIdx.x % T, n = (int)a.in.n;
    const float inv_n = 1.f / (float)n;
    f32x4 w[V4], sum_w[V4], sum_b[V4];
#pragma unroll
    for (int k = 0; k < V4; ++k) w[k] = f32x4{1.f, 1.f, 1.f, 1.f}, sum_w[k] = sum_b[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.weight) load_row<T, V4>(w, a.weight, n, t);
    int turn = 0;
    f32x4 next_x[V4], next_dy[V4];
    float next_mean = 0.f, next_rstd = 0.f;
    auto load = [&](int64_t row) {
        load_row<T, V4>(next_x, norm_row(a.in, row), n, t);
        load_row<T, V4>(next_dy, a.dy + row * a.in.n, n, t); // zero behind the last column
        next_mean = a.mean[row];
        next_rstd = a.rstd[row];
    };
    const int64_t first = (int64_t)blockIdx.x * R + threadIdx.x / T, stride = a.row_groups * R;
    if (AHEAD && first < a.in.rows) load(first);
    for (int64_t row = first; row < a.in.rows; row += stride, turn ^= 1) {
        if (!AHEAD) load(row);
        f32x4 x[V4], dy[V4];
#pragma unroll
        for (int k = 0; k < V4; ++k) x[k] = next_x[k], dy[k] = next_dy[k];
        const float mean = next_mean, rstd = next_rstd;
        if (AHEAD && row + stride < a.in.rows) load(row + stride);
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int k = 0; k < V4; ++k) {
            x[k] = (x[k] - mean) * rstd;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * (t + T * k) + e >= n) x[k][e] = 0.f;
            sum_w[k] += dy[k] * x[k];
            sum_b[k] += dy[k];
            dy[k] *= w[k];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c1 += dy[k][e];
                c2 += dy[k][e] * x[k][e];
            }
        }
        if (!a.grad_x) continue; // the same in every thread
        c1 = group_sum<W>(c1, slots[turn][0]) * inv_n;
        c2 = group_sum<W>(c2, slots[turn][1]) * inv_n;
#pragma unroll
        for (int k = 0; k < V4; ++k) x[k] = rstd * (dy[k] - c1 - x[k] * c2);
        float* g = a.grad_x + row * a.in.n;
        if (a.accumulate) {
            load_row<T, V4>(dy, g, n, t);
#pragma unroll
            for (int k = 0; k < V4; ++k) x[k] += dy[k];
        }
        store_row<T, V4>(g, x, n, t);
    }
    if (!a.partial) return;
    float* to = a.partial + 2 * (int64_t)blockIdx.x * a.in.n;
    if constexpr (W == 4) {
        store_row<T, V4>(to, sum_w, n, t);
        store_row<T, V4>(to + a.in.n, sum_b, n, t);
    } else { // the workgroup's four rows of sums are one
        __shared__ f32x4 sums[4][2][64 * V4];
#pragma unroll
        for (int k = 0; k < V4; ++k) sums[threadIdx.x / T][0][t + T * k] = sum_w[k], sums[threadIdx.x / T][1][t + T * k] = sum_b[k];
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * 64 * V4; c += 256) {
            const int which = c / (64 * V4), g = c - which * 64 * V4;
            const f32x4 s = (sums[0][which][g] + sums[1][which][g]) + (sums[2][which][g] + sums[3][which][g]);
            for (int e = 0; e < 4; ++e)
                if (4 * g + e < n) to[which * a.in.n + 4 * g + e] = s[e];
        }
    }
}

__global__ __launch_bounds__(256) void norm_backward_any_kernel(const NormBackward a) { // grad_x alone
    __shared__ float slots[2][4];
    const int64_t n = a.in.n, cs = a.in.col_stride;
    for (int64_t row = blockIdx.x; row < a.in.rows; row += gridDim.x) {
        const float* __restrict p = norm_row(a.in, row);
        const float* __restrict dy = a.dy + row * n;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float c1 = 0.f, c2 = 0.f;
        for (int64_t c = threadIdx.x; c < n; c += 256) {
            const float g = dy[c] * (a.weight ? a.weight[c] : 1.f);
            c1 += g;
            c2 += g * ((p[c * cs] - mean) * rstd);
        }
        c1 = group_sum<4>(c1, slots[0]) / (float)n;
        c2 = group_sum<4>(c2, slots[1]) / (float)n;
        for (int64_t c = threadIdx.x; c < n; c += 256) {
            const float g = dy[c] * (a.weight ? a.weight[c] : 1.f);
            const float d = rstd * (g - c1 - (p[c * cs] - mean) * rstd * c2);
            a.grad_x[row * n + c] = a.accumulate ? a.grad_x[row * n + c] + d : d;
        }
    }
}

// partial sums of a run of rows for 256 columns: the form without registers for a row
__global__ __launch_bounds__(256) void norm_columns_any_kernel(const NormBackward a) {
    const int64_t n = a.in.n, c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t per = (a.in.rows + a.parts - 1) / a.parts;
    const int64_t lo = (int64_t)blockIdx.y * per, hi = lo + per < a.in.rows ? lo + per : a.in.rows;
    if (c >= n) return;
    float sw = 0.f, sb = 0.f;
    for (int64_t row = lo; row < hi; ++row) {
        const float g = a.dy[row * n + c];
        sw += g * ((norm_row(a.in, row)[c * a.in.col_stride] - a.mean[row]) * a.rstd[row]);
        sb += g;
    }
    a.partial[2 * (int64_t)blockIdx.y * n + c] = sw;
    a.partial[(2 * (int64_t)blockIdx.y + 1) * n + c] = sb;
}

// The parts of 64 columns of dw or db added up: each of the 16 wavefronts takes every 16th part, then their sums are added in order.
__global__ __launch_bounds__(1024) void norm_join_kernel(const NormBackward a) {
    __shared__ float s[16][64];
    const int64_t n = a.in.n, c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int which = blockIdx.y, wave = threadIdx.x >> 6;
    float* out = which ? a.grad_bias : a.grad_weight;
    if (!out) return; // the same in the whole workgroup
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < n) {
        const float* __restrict p = a.partial + which * n + c;
        int64_t i = wave;
        for (; i + 112 < a.parts; i += 128) // eight loads in flight
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] += p[2 * (i + 16 * u) * n];
        for (; i < a.parts; i += 16) v[0] += p[2 * i * n];
    }
    s[wave][threadIdx.x & 63] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    __syncthreads();
    if (wave == 0 && c < n) {
        float sum = s[0][threadIdx.x];
        for (int w = 1; w < 16; ++w) sum += s[w][threadIdx.x];
        out[c] = a.accumulate ? out[c] + sum : sum;
    }
}

constexpr int64_t kMostColumns = 1 << 27;

int norm_rows(const tenmo_view* X, const char* who, NormRows* r) {
    if (int rc = check_operand(X, 1, TENMO_MAX_RANK, who, "X")) return rc;
    r->n = X->shape[X->rank - 1];
    if (r->n < 1) return refuse(TENMO_ERR_INVALID_SHAPE, "%s: the last axis is empty", who);
    r->rows = elements(X) / r->n;
    r->col_stride = X->strides[X->rank - 1];
    r->x = X->data ? X->data + X->offset : nullptr;
    r->rank = 0;
    for (int d = 0; d < X->rank - 1; ++d) { // axes that continue the one before them are one axis
        if (X->shape[d] == 1) continue;
        if (r->rank && r->stride[r->rank - 1] == X->shape[d] * X->strides[d]) {
            r->shape[r->rank - 1] *= X->shape[d];
            r->stride[r->rank - 1] = X->strides[d];
        } else {
            r->shape[r->rank] = X->shape[d];
            r->stride[r->rank++] = X->strides[d];
        }
    }
    if (r->n > kMostColumns) return refuse(TENMO_ERR_UNSUPPORTED, "%s: more than 2^27 columns", who);
    return 0;
}

// Whether the n floats at p may share a place with the view
bool may_share(const float* p, int64_t n, const tenmo_view* X) {
    int64_t low = X->offset, high = X->offset;
    for (int d = 0; d < X->rank; ++d) (X->strides[d] < 0 ? low : high) += (X->shape[d] - 1) * X->strides[d];
    return p && (uintptr_t)p <= (uintptr_t)(X->data + high) && (uintptr_t)(X->data + low) < (uintptr_t)(p + n);
}

// Rows of partial sums, which is workgroups: enough to fill the chip two or three times over
constexpr int64_t kNormWorkgroups = 768;
int64_t norm_rows_at_a_time(int64_t n) { return n <= 1024 ? 4 : 1; }
int64_t norm_parts(int64_t rows, int64_t n) { return std::max<int64_t>(1, std::min<int64_t>((rows + norm_rows_at_a_time(n) - 1) / norm_rows_at_a_time(n), kNormWorkgroups)); }

// Few rows: dw and db by workgroups of their own in the same launch, which read x and dy again, instead of a launch behind it (a backward call of 256 rows of 768: 14.6 us, 17.9 with the
// join; [1024, 768] 14.0 and 17.7, [2048, 768] 36.7 and 30.6 waited for, [512, 8000] 45.7 and 43.2).
bool norm_columns_in_launch(int64_t rows, int64_t n) { return rows <= 1024 && rows * n <= 1 << 21; }

// a workgroup a row, or four, up to what a launch may hold; beyond that they take further ones
unsigned norm_grid(int64_t groups) { return (unsigned)std::min<int64_t>(groups, 1 << 22); }

template <class Args>
using NormKernel = void (*)(Args);

// by the groups of 4 columns that a thread holds: of 64 threads, or of 256
#define TENMO_NORM_FOR(kernel)                                                                                                                                     \
    switch (n <= 1024 ? (n + 255) / 256 : 4 + (n + 1023) / 1024) {                                                                                                 \
        case 1: return kernel<1, 1>;                                                                                                                               \
        case 2: return kernel<1, 2>;                                                                                                                               \
        case 3: return kernel<1, 3>;                                                                                                                               \
        case 4: return kernel<1, 4>;                                                                                                                               \
        case 6: return kernel<4, 2>;                                                                                                                               \
        case 7: return kernel<4, 3>;                                                                                                                               \
        case 8: return kernel<4, 4>;                                                                                                                               \
        case 9:                                                                                                                                                    \
        case 10: return kernel<4, 6>;                                                                                                                              \
        default: return kernel<4, 8>;                                                                                                                              \
    }
NormKernel<const NormForward> norm_forward_for(int64_t n) { TENMO_NORM_FOR(norm_forward_kernel) }
NormKernel<const NormBackward> norm_backward_for(int64_t n) { TENMO_NORM_FOR(norm_backward_kernel) }
#undef TENMO_NORM_FOR

} // namespace
} // namespace tenmo

using namespace tenmo;

extern "C" {

int tenmo_hip_layer_norm_forward_f32(const tenmo_view* X, const float* weight, const float* bias, float eps, float* out, float* mean, float* rstd, int32_t sync) {
    const char* who = "tenmo_hip_layer_norm_forward_f32";
    NormForward a{};
    if (int rc = norm_rows(X, who, &a.in)) return rc;
    if (!(eps >= 0.f)) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: eps must not be negative, got %g", who, (double)eps);
    if (!mean != !rstd) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: mean and rstd are wanted together or not at all", who);
    if (a.in.rows > 0 && !out) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: null out", who);
    Call call(who);
    if (int rc = call.begin()) return rc;
    if (a.in.rows == 0) return 0;
    a.weight = weight; a.bias = bias; a.eps = eps; a.out = out; a.mean = mean; a.rstd = rstd;
    if (a.in.n <= 8192 && (a.in.col_stride == 1 || a.in.n == 1)) {
        const int64_t rows_at_a_time = norm_rows_at_a_time(a.in.n);
        hipLaunchKernelGGL(norm_forward_for(a.in.n), dim3(norm_grid((a.in.rows + rows_at_a_time - 1) / rows_at_a_time)), dim3(256), 0, call.state.stream, a);
    } else {
        hipLaunchKernelGGL(norm_forward_any_kernel, dim3(norm_grid(a.in.rows)), dim3(256), 0, call.state.stream, a);
    }
    return call.finish(sync);
}

int64_t tenmo_hip_layer_norm_backward_workspace_bytes(int64_t rows, int64_t n) {
    const char* who = "tenmo_hip_layer_norm_backward_workspace_bytes";
    if (rows < 0 || n < 1) return refuse(TENMO_ERR_INVALID_SHAPE, "%s: needs rows >= 0 and columns >= 1", who);
    if (n > kMostColumns) return refuse(TENMO_ERR_UNSUPPORTED, "%s: more than 2^27 columns", who);
    if (rows == 0) return 0;
    Workspace ws(nullptr, 0);
    ws.take<float>(2 * norm_parts(rows, n) * n);
    return ws.used();
}

int tenmo_hip_layer_norm_backward_f32(const tenmo_view* X, const float* weight, const float* mean, const float* rstd, const float* dY,
                                      float* grad_X, float* grad_weight, float* grad_bias, int32_t accumulate,
                                      void* workspace, int64_t workspace_bytes, int32_t sync) {
    const char* who = "tenmo_hip_layer_norm_backward_f32";
    NormBackward a{};
    if (int rc = norm_rows(X, who, &a.in)) return rc;
    if (a.in.rows > 0 && (!mean || !rstd || !dY)) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    Call call(who);
    if (int rc = call.begin()) return rc;
    if (!grad_X && !grad_weight && !grad_bias) return 0;
    a.weight = weight; a.mean = mean; a.rstd = rstd; a.dy = dY;
    a.grad_x = grad_X; a.grad_weight = grad_weight; a.grad_bias = grad_bias; a.accumulate = accumulate ? 1 : 0;
    const hipStream_t stream = call.state.stream;
    const int64_t n = a.in.n;
    const int64_t all = a.in.rows * n;
    const bool in_place = all > 0 && (may_share(grad_X, all, X) || (grad_X && (uintptr_t)grad_X < (uintptr_t)(dY + all) && (uintptr_t)dY < (uintptr_t)(grad_X + all)));
    const bool by_rows = n <= 8192 && (a.in.col_stride == 1 || n == 1);
    const bool columns_too = by_rows && all > 0 && !in_place && norm_columns_in_launch(a.in.rows, n) && (grad_weight || grad_bias);
    if ((grad_weight || grad_bias) && !columns_too) {
        Workspace ws(workspace, workspace_bytes);
        a.parts = a.in.rows ? norm_parts(a.in.rows, n) : 0;
        a.partial = ws.take<float>(2 * a.parts * n);
        if (int rc = ws.check(who)) return rc;
    }
    if (a.in.rows > 0) {
        if (by_rows) {
            a.row_groups = grad_X || !columns_too ? norm_parts(a.in.rows, n) : 0;
            hipLaunchKernelGGL(norm_backward_for(n), dim3((unsigned)(a.row_groups + (columns_too ? (n + 15) / 16 : 0))), dim3(256), 0, stream, a);
        } else {
            // (the sums first: grad_X may be written where they read)
            if (a.partial) hipLaunchKernelGGL(norm_columns_any_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)a.parts), dim3(256), 0, stream, a);
            if (grad_X) hipLaunchKernelGGL(norm_backward_any_kernel, dim3(norm_grid(a.in.rows)), dim3(256), 0, stream, a);
        }
    }
    if ((grad_weight || grad_bias) && !columns_too) hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)((n + 63) / 64), 2), dim3(1024), 0, stream, a);
    return call.finish(sync);
}

} // extern "C"
