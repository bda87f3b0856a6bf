// Attention for few query rows and short sequences.
//
// Forward: one new token of each sequence, or a handful, against a long run of keys.
//
//   m = max_j s_j,  l = sum_j exp(s_j - m),  o = sum_j exp(s_j - m) v_j / l,   s_j = scale q . k_j
//
// Bound: HBM, every key and value once (8 D bytes a key and key head); the arithmetic is 4 D flop a row.
//   * the query rows that share a key head (heads of its group x queries) are worked on together, up to R of them, so that a key is
//     read once for all of them.
//   * a key's D values lie across L lanes, 4 in each (16-byte loads, L = 8, 16, 32 for D up to 32, 64, 128); the 64 / L key slots of a
//     wavefront each keep a running maximum and sum of their own, so that nothing crosses a slot before the end.  Each slot takes U keys at
//     a time: U independent loads of K and of V in flight a lane, one rescaling for the U.
//   * the keys of a sequence are cut into `splits` runs when there are too few (sequence, key head) pairs to fill the chip; the runs' maxima, sums
//     and outputs are joined by a second launch in a fixed order.
#include "attention.hpp"

#include <algorithm>

namespace tenmo {
namespace {

struct RowsArgs {
    AttnShape s;
    AttnOperand q, k, v;
    float *out, *lse;
    float* part; // [splits][batch][heads][queries][dim + 2]: the run's o (not divided), its maximum and its sum; NULL with one run
    int splits, row_blocks;
};

template <int L, int R, int KIND> // lanes a key, rows a workgroup, how rows are loaded
__global__ __launch_bounds__(256) void attn_rows_kernel(const RowsArgs a) {
    constexpr int SLOTS = 64 / L, U = R > 4 ? 2 : 4;
    __shared__ float join_m[4][SLOTS][R], join_l[4][SLOTS][R];
    __shared__ f32x4 join_o[4][SLOTS][R][L];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = lane / L, part = lane % L, D = a.s.dim;
    int rest = blockIdx.x;
    const int split = rest % a.splits; rest /= a.splits;
    const int rb = rest % a.row_blocks; rest /= a.row_blocks;
    const int hk = rest % a.s.kv_heads, b = rest / a.s.kv_heads;
    const int length = attn_length(a.s, b), start = attn_start(a.s, b);
    const int rows = a.s.group * a.s.queries; // row r: head hk * group + r / queries, query r % queries
    const int row0 = rb * R;

    f32x4 q[R];
    int limit[R], least = length, most = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + r < rows ? row0 + r : rows - 1;
        const int h = hk * a.s.group + row / a.s.queries, i = row % a.s.queries;
        q[r] = attn_load4<KIND>(a.q.p + b * a.q.b + i * a.q.s + h * a.q.h, a.q.d, part, D) * a.s.scale;
        limit[r] = attn_limit(length, start, i);
        least = limit[r] < least ? limit[r] : least;
        most = limit[r] > most ? limit[r] : most;
    }
    // this run's keys
    const int per = (most + a.splits - 1) / a.splits;
    const int lo = split * per < most ? split * per : most, hi = lo + per < most ? lo + per : most;

    float m[R], l[R];
    f32x4 o[R];
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = kNone, l[r] = 0.f, o[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* kp = a.k.p + b * a.k.b + hk * a.k.h;
    const float* vp = a.v.p + b * a.v.b + hk * a.v.h;
    for (int j0 = lo + wave * SLOTS + slot; __any(j0 < hi); j0 += 4 * SLOTS * U) {
        f32x4 k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) { // a slot without a key of its own reads the run's last one and does not use it
            const int64_t j = j0 + 4 * SLOTS * u < hi ? j0 + 4 * SLOTS * u : hi - 1;
            k[u] = attn_load4<KIND>(kp + j * a.k.s, a.k.d, part, D);
            v[u] = attn_load4<KIND>(vp + j * a.v.s, a.v.d, part, D);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float s[U], top = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float x = lanes_sum<L>(dot4(q[r], k[u]));
                const int j = j0 + 4 * SLOTS * u;
                s[u] = j < hi && j < limit[r] ? x : kNone;
                top = fmaxf(top, s[u]);
            }
            const float keep = below(m[r], top);
            m[r] = top;
            l[r] *= keep;
            o[r] *= keep;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + 4 * SLOTS * u;
                if (j >= hi || j >= limit[r]) continue; // its value may be anything
                const float p = below(s[u], top);
                l[r] += p;
                o[r] += p * v[u];
            }
        }
    }
    // the slots of the workgroup, added in order
#pragma unroll
    for (int r = 0; r < R; ++r) {
        join_o[wave][slot][r][part] = o[r];
        if (part == 0) join_m[wave][slot][r] = m[r], join_l[wave][slot][r] = l[r];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < R * L; x += 256) {
        const int r = x / L, c = x % L;
        if (row0 + r >= rows) continue;
        float top = kNone, sum = 0.f;
        for (int w = 0; w < 4; ++w)
            for (int t = 0; t < SLOTS; ++t) top = fmaxf(top, join_m[w][t][r]);
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < 4; ++w)
            for (int t = 0; t < SLOTS; ++t) {
                const float keep = below(join_m[w][t][r], top);
                sum += keep * join_l[w][t][r];
                acc += keep * join_o[w][t][r][c];
            }
        const int h = hk * a.s.group + (row0 + r) / a.s.queries, i = (row0 + r) % a.s.queries;
        const int64_t row = ((int64_t)b * a.s.heads + h) * a.s.queries + i;
        float* to;
        if (a.part) {
            to = a.part + ((int64_t)split * a.s.batch * a.s.heads * a.s.queries + row) * (D + 2);
            if (c == 0) to[D] = top, to[D + 1] = sum;
        } else {
            to = a.out + (((int64_t)b * a.s.queries + i) * a.s.heads + h) * D;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            acc = sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : acc * inv;
            if (c == 0 && a.lse) a.lse[row] = sum == 0.f ? kNone : top + logf(sum);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * c + e < D) to[4 * c + e] = acc[e];
    }
}

// The runs of one row joined: W wavefronts, each with every W-th run, two values of d a lane.
template <int W>
__global__ __launch_bounds__(64 * W) void attn_join_kernel(const AttnShape s, const float* __restrict part, int splits, float* __restrict out, float* __restrict lse) {
    __shared__ float keep_of[kMostRuns], sum_of[kMostRuns], slots[2][W], o_of[W][128];
    const int D = s.dim, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x, pitch = (int64_t)s.batch * s.heads * s.queries * (D + 2);
    const float* __restrict p = part + row * (D + 2);
    float top = kNone;
    for (int t = threadIdx.x; t < splits; t += 64 * W) {
        keep_of[t] = p[t * pitch + D];
        sum_of[t] = p[t * pitch + D + 1];
        top = fmaxf(top, keep_of[t]);
    }
    top = wave_max(top);
    if (lane == 0) slots[0][wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, slots[0][w]);
    float sum = 0.f;
    for (int t = threadIdx.x; t < splits; t += 64 * W) {
        const float keep = below(keep_of[t], top);
        sum += keep * sum_of[t];
        keep_of[t] = keep;
    }
    sum = group_sum<W>(sum, slots[1]); // (a barrier: keep_of is whole)
    float o[2] = {0.f, 0.f};
#pragma unroll 8
    for (int t = wave; t < splits; t += W)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (lane + 64 * e < D) o[e] += keep_of[t] * p[t * pitch + lane + 64 * e];
    o_of[wave][lane] = o[0];
    o_of[wave][lane + 64] = o[1];
    __syncthreads();
    const int i = (int)(row % s.queries), h = (int)(row / s.queries % s.heads), d = threadIdx.x;
    const int64_t b = row / s.queries / s.heads;
    if (d < D) {
        float x = o_of[0][d];
        for (int w = 1; w < W; ++w) x += o_of[w][d];
        out[((b * s.queries + i) * s.heads + h) * D + d] = sum == 0.f ? 0.f : x / sum;
    }
    if (d == 0 && lse) lse[row] = sum == 0.f ? kNone : top + logf(sum);
}

int kind_of(const AttnOperand& q, const AttnOperand& k, const AttnOperand& v, int D) { return attn_kind(q.d == 1 && k.d == 1 ? v.d : 0, D); }

template <int L, int R>
void launch_rows(const RowsArgs& a, unsigned grid, hipStream_t stream) {
    const int kind = kind_of(a.q, a.k, a.v, a.s.dim);
    if (kind == kLoadWhole) hipLaunchKernelGGL((attn_rows_kernel<L, R, kLoadWhole>), dim3(grid), dim3(256), 0, stream, a);
    else if (kind == kLoadTail) hipLaunchKernelGGL((attn_rows_kernel<L, R, kLoadTail>), dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attn_rows_kernel<L, R, kLoadAny>), dim3(grid), dim3(256), 0, stream, a);
}
template <int L>
void launch_rows(const RowsArgs& a, int r, unsigned grid, hipStream_t stream) {
    if (r == 1) launch_rows<L, 1>(a, grid, stream);
    else if (r <= 4) launch_rows<L, 4>(a, grid, stream);
    else launch_rows<L, 8>(a, grid, stream);
}

// Backward: s and dP = dout . v again for each allowed pair, p = exp(s - lse), dS = p (dP - delta) with delta = dout . out; dq = scale sum_j dS k_j over a row's keys,
// dv_j = sum_i p_ij dout_i and dk_j = scale sum_i dS_ij q_i over the queries of the heads that share a key's.  What bounds it at the sizes it is taken for is latency, so both are one launch: the
// blocks of keys work delta out of out again (a call of [2,33,4,32]: 17.7 us, 21.9 in two launches; [1,128,8,128]: 19.2, 28.4).
struct RowsBackward {
    AttnBackward b;
    int key_blocks;  // of a key head
    int key_groups;  // workgroups of keys, before those of rows
};

__device__ __forceinline__ void add_to(const AttnOperand& g, int64_t at, int part, int D, f32x4 x, int accumulate) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (4 * part + e < D) {
            float* to = g.p + at + (4 * part + e) * g.d;
            *to = accumulate ? *to + x[e] : x[e];
        }
}

template <int L, int KIND>
__device__ __forceinline__ void rows_dq(const RowsBackward& a, int id) { // a wavefront a row
    constexpr int SLOTS = 64 / L, U = 2;
    const AttnShape& s = a.b.s;
    const int lane = threadIdx.x & 63, slot = lane / L, part = lane % L, D = s.dim;
    const int64_t row = (int64_t)id * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)s.batch * s.heads * s.queries) return;
    const int i = (int)(row % s.queries), h = (int)(row / s.queries % s.heads), b = (int)(row / s.queries / s.heads), hk = h / s.group;
    const int limit = attn_limit(attn_length(s, b), attn_start(s, b), i);
    const int64_t dense = (((int64_t)b * s.queries + i) * s.heads + h) * D;
    const f32x4 q = attn_load4<KIND>(a.b.q.p + b * a.b.q.b + i * a.b.q.s + h * a.b.q.h, a.b.q.d, part, D) * s.scale;
    const f32x4 g = attn_load4<KIND>(a.b.dout + dense, 1, part, D), o = attn_load4<KIND>(a.b.out + dense, 1, part, D);
    const float delta = lanes_sum<L>(dot4(g, o)), lse = a.b.lse[row];
    const float* kp = a.b.k.p + b * a.b.k.b + hk * a.b.k.h;
    const float* vp = a.b.v.p + b * a.b.v.b + hk * a.b.v.h;
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int j0 = slot; __any(j0 < limit); j0 += SLOTS * U) {
        f32x4 k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = j0 + SLOTS * u < limit ? j0 + SLOTS * u : limit - 1;
            k[u] = attn_load4<KIND>(kp + j * a.b.k.s, a.b.k.d, part, D);
            v[u] = attn_load4<KIND>(vp + j * a.b.v.s, a.b.v.d, part, D);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float x = lanes_sum<L>(dot4(q, k[u])), dp = lanes_sum<L>(dot4(g, v[u]));
            if (j0 + SLOTS * u < limit) acc += __expf(x - lse) * (dp - delta) * k[u];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = L; d < 64; d <<= 1) acc[e] += __shfl_xor(acc[e], d, 64);
    if (slot == 0) add_to(a.b.grad_q, b * a.b.grad_q.b + i * a.b.grad_q.s + h * a.b.grad_q.h, part, D, acc * s.scale, a.b.accumulate);
}

// a slot a key, the queries dealt to the 4 wavefronts, four of each at a time
template <int L, int KIND>
__device__ __forceinline__ void rows_dkv(const RowsBackward& a, int id) {
    constexpr int SLOTS = 64 / L, U = 4;
    __shared__ f32x4 join[2][4][SLOTS][L];
    const AttnShape& s = a.b.s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = lane / L, part = lane % L, D = s.dim;
    int rest = id;
    const int j = rest % a.key_blocks * SLOTS + slot; rest /= a.key_blocks;
    const int hk = rest % s.kv_heads, b = rest / s.kv_heads;
    const int length = attn_length(s, b), start = attn_start(s, b);
    const int64_t jr = j < s.keys ? j : s.keys - 1;
    const f32x4 k = attn_load4<KIND>(a.b.k.p + b * a.b.k.b + hk * a.b.k.h + jr * a.b.k.s, a.b.k.d, part, D);
    const f32x4 v = attn_load4<KIND>(a.b.v.p + b * a.b.v.b + hk * a.b.v.h + jr * a.b.v.s, a.b.v.d, part, D);
    f32x4 dk{0.f, 0.f, 0.f, 0.f}, dv = dk;
    // the first query that sees the first of these keys
    const int first = j - slot < length ? (j - slot > start ? j - slot - start : 0) : s.queries;
    for (int h = hk * s.group; h < (hk + 1) * s.group; ++h)
        for (int i0 = first + wave; i0 < s.queries; i0 += 4 * U) {
            f32x4 q[U], g[U], o[U];
            float lse[U];
#pragma unroll
            for (int u = 0; u < U; ++u) { // (the last query again where there is none)
                const int i = i0 + 4 * u < s.queries ? i0 + 4 * u : s.queries - 1;
                const int64_t row = ((int64_t)b * s.heads + h) * s.queries + i;
                q[u] = attn_load4<KIND>(a.b.q.p + b * a.b.q.b + i * a.b.q.s + h * a.b.q.h, a.b.q.d, part, D);
                const int64_t dense = (((int64_t)b * s.queries + i) * s.heads + h) * D;
                g[u] = attn_load4<KIND>(a.b.dout + dense, 1, part, D);
                o[u] = attn_load4<KIND>(a.b.out + dense, 1, part, D);
                lse[u] = a.b.lse[row];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 4 * u;
                const float x = lanes_sum<L>(dot4(q[u], k)) * s.scale, dp = lanes_sum<L>(dot4(g[u], v)), delta = lanes_sum<L>(dot4(g[u], o[u]));
                if (i >= s.queries || j >= attn_limit(length, start, i)) continue; // its row may hold anything
                const float p = __expf(x - lse[u]);
                dv += p * g[u];
                dk += p * (dp - delta) * q[u];
            }
        }
    join[0][wave][slot][part] = dk;
    join[1][wave][slot][part] = dv;
    __syncthreads();
    if (wave != 0 || j >= s.keys) return;
    dk = (join[0][0][slot][part] + join[0][1][slot][part]) + (join[0][2][slot][part] + join[0][3][slot][part]);
    dv = (join[1][0][slot][part] + join[1][1][slot][part]) + (join[1][2][slot][part] + join[1][3][slot][part]);
    if (a.b.grad_k.p) add_to(a.b.grad_k, b * a.b.grad_k.b + j * a.b.grad_k.s + hk * a.b.grad_k.h, part, D, dk * s.scale, a.b.accumulate);
    if (a.b.grad_v.p) add_to(a.b.grad_v, b * a.b.grad_v.b + j * a.b.grad_v.s + hk * a.b.grad_v.h, part, D, dv, a.b.accumulate);
}

template <int L, int KIND>
__global__ __launch_bounds__(256) void attn_rows_backward_kernel(const RowsBackward a) {
    if ((int)blockIdx.x < a.key_groups) rows_dkv<L, KIND>(a, blockIdx.x);
    else rows_dq<L, KIND>(a, blockIdx.x - a.key_groups);
}

template <int L>
void launch_rows_backward(const RowsBackward& a, unsigned grid, hipStream_t stream) {
    const int kind = kind_of(a.b.q, a.b.k, a.b.v, a.b.s.dim);
    if (kind == kLoadWhole) hipLaunchKernelGGL((attn_rows_backward_kernel<L, kLoadWhole>), dim3(grid), dim3(256), 0, stream, a);
    else if (kind == kLoadTail) hipLaunchKernelGGL((attn_rows_backward_kernel<L, kLoadTail>), dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attn_rows_backward_kernel<L, kLoadAny>), dim3(grid), dim3(256), 0, stream, a);
}

} // namespace

void attn_rows_backward(const AttnBackward& b, hipStream_t stream) {
    RowsBackward a{};
    a.b = b;
    const int slots = b.s.dim <= 32 ? 8 : b.s.dim <= 64 ? 4 : 2;
    a.key_blocks = (b.s.keys + slots - 1) / slots;
    a.key_groups = b.grad_k.p || b.grad_v.p ? b.s.batch * b.s.kv_heads * a.key_blocks : 0;
    const int row_groups = b.grad_q.p ? (int)(((int64_t)b.s.batch * b.s.heads * b.s.queries + 3) / 4) : 0;
    const unsigned grid = (unsigned)(a.key_groups + row_groups);
    if (b.s.dim <= 32) launch_rows_backward<8>(a, grid, stream);
    else if (b.s.dim <= 64) launch_rows_backward<16>(a, grid, stream);
    else launch_rows_backward<32>(a, grid, stream);
}

void attn_rows_forward(const AttnShape& s, const AttnOperand& q, const AttnOperand& k, const AttnOperand& v, float* out, float* lse,
                       Workspace& ws, int cus, hipStream_t stream, bool launch) {
    RowsArgs a{};
    a.s = s; a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse;
    const int rows = s.group * s.queries, r = rows == 1 ? 1 : rows <= 4 ? 4 : 8;
    a.row_blocks = (rows + r - 1) / r;
    const int64_t groups = (int64_t)s.batch * s.kv_heads * a.row_blocks;
    // four workgroups a CU fill it (16 wavefronts); a run of fewer than 128 keys is not worth its part of the join
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>((4LL * cus + groups - 1) / groups, std::min(s.keys / 128, kMostRuns)));
    if (a.splits > 1) a.part = ws.take<float>((int64_t)a.splits * s.batch * s.heads * s.queries * (s.dim + 2));
    if (!launch) return;
    const unsigned grid = (unsigned)(groups * a.splits);
    if (s.dim <= 32) launch_rows<8>(a, r, grid, stream);
    else if (s.dim <= 64) launch_rows<16>(a, r, grid, stream);
    else launch_rows<32>(a, r, grid, stream);
    if (a.splits > 1) attn_join(s, a.part, a.splits, out, lse, stream);
}

void attn_join(const AttnShape& s, const float* part, int splits, float* out, float* lse, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)s.batch * s.heads * s.queries));
    // many runs of few rows: one load of each wavefront's runs after another is what takes the time (128 runs of 32 rows: 19 us with 4 wavefronts)
    if (splits > 16) hipLaunchKernelGGL(attn_join_kernel<16>, grid, dim3(1024), 0, stream, s, part, splits, out, lse);
    else hipLaunchKernelGGL(attn_join_kernel<4>, grid, dim3(256), 0, stream, s, part, splits, out, lse);
}

} // namespace tenmo
