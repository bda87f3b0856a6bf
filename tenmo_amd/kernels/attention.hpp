// What the kernels of attention share: the operands, and which keys a query may use.
#ifndef TENMO_KERNELS_ATTENTION_HPP
#define TENMO_KERNELS_ATTENTION_HPP
#include "entry.hpp"

namespace tenmo {

struct AttnOperand { // element (b, s, h, d)
    float* p;
    int64_t b, s, h, d;
};

struct AttnShape {
    int batch, queries, keys, heads, kv_heads, dim;
    int group;   // heads / kv_heads
    int causal;
    float scale;
    const int32_t *key_lengths, *query_starts;
};

// keys of sequence b
__device__ __forceinline__ int attn_length(const AttnShape& a, int b) {
    const int n = a.key_lengths ? a.key_lengths[b] : a.keys;
    return n < 0 ? 0 : n > a.keys ? a.keys : n;
}
// position of the first query of sequence b, limited to where it makes a difference (so that sums with an index stay in 32 bits)
__device__ __forceinline__ int attn_start(const AttnShape& a, int b) {
    if (!a.causal) return a.keys;
    const int s = a.query_starts ? a.query_starts[b] : a.keys - a.queries;
    return s < -a.queries ? -a.queries : s > a.keys ? a.keys : s;
}
// query i may use the keys 0 .. attn_limit - 1 (i >= 0)
__device__ __forceinline__ int attn_limit(int length, int start, int i) {
    const int64_t n = (int64_t)start + i + 1;
    return n < 0 ? 0 : n < length ? (int)n : length;
}

constexpr float kNone = -__builtin_inff(); // the maximum and the logarithm of the sum of no scores

// exp(a - m) for a running maximum m >= a, which is -inf while nothing was seen.  The hardware's 2^x after one multiplication: x below the
// maximum by t comes out with a relative error of (t + 2) 2^-24, where its weight is exp(-t).
__device__ __forceinline__ float below(float a, float m) { return __expf(a - (m == kNone ? 0.f : m)); }

// Four values of d of a row, of which the first is 4 * part; zero behind the last.  Three ways, none with a branch of a lane's own: where lanes part, each waits for the loads that the others
// have under way.  What a lane has no values for it reads at the row's end and drops.
enum { kLoadAny, kLoadWhole, kLoadTail }; // any stride; adjacent values, a multiple of four of them; adjacent values, four at least
__device__ __host__ __forceinline__ int attn_kind(int64_t d, int D) { return d != 1 || D < 4 ? kLoadAny : D % 4 ? kLoadTail : kLoadWhole; }
template <int KIND>
__device__ __forceinline__ f32x4 attn_load4(const float* row, int64_t ds, int part, int D) {
    const int at = 4 * part;
    f32x4 x;
    if (KIND == kLoadWhole) {
        x = *(const f32x4_u*)(row + (at < D ? at : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = at < D ? x[e] : 0.f;
    } else if (KIND == kLoadTail) { // the last group is read with values of the one before it, and moved down
        x = *(const f32x4_u*)(row + (at < D - 4 ? at : D - 4));
        const int by = at - (D - 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y = by <= 0 ? x[e] : 0.f;
#pragma unroll
            for (int f = e + 1; f < 4; ++f) y = by == f - e ? x[f] : y;
            x[e] = y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = row[(at + e < D ? at + e : D - 1) * ds];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = at + e < D ? x[e] : 0.f;
    }
    return x;
}
template <int KIND> struct LoadKind { static constexpr int value = KIND; };
// f with the kind as a constant: one branch, that all lanes take together, around all loads of a kind
template <class F>
__device__ __forceinline__ void attn_with_kind(int kind, F f) {
    if (kind == kLoadWhole) f(LoadKind<kLoadWhole>{});
    else if (kind == kLoadTail) f(LoadKind<kLoadTail>{});
    else f(LoadKind<kLoadAny>{});
}
__device__ __forceinline__ float dot4(f32x4 a, f32x4 b) { return (a[0] * b[0] + a[1] * b[1]) + (a[2] * b[2] + a[3] * b[3]); }
struct AttnBackward {
    AttnShape s;
    AttnOperand q, k, v;           // q.p .. never written
    AttnOperand grad_q, grad_k, grad_v; // p NULL: not wanted
    const float *out, *lse, *dout;
    int accumulate;
};

// ---- attention_rows.hip ----
void attn_rows_forward(const AttnShape&, const AttnOperand& q, const AttnOperand& k, const AttnOperand& v, float* out, float* lse,
                       Workspace& ws, int cus, hipStream_t stream, bool launch);

void attn_rows_backward(const AttnBackward&, hipStream_t stream); // needs no workspace
constexpr int kMostRuns = 1024;
// joins `splits` runs of keys: part [splits][batch][heads][queries][dim + 2] holds each run's sum of p v, its maximum and its sum of p
void attn_join(const AttnShape&, const float* part, int splits, float* out, float* lse, hipStream_t stream);

// ---- attention_tiles.hip ----
void attn_tiles_forward(const AttnShape&, const AttnOperand& q, const AttnOperand& k, const AttnOperand& v, float* out, float* lse,
                        Workspace& ws, int cus, hipStream_t stream, bool launch);
void attn_tiles_backward(const AttnBackward&, Workspace& ws, int cus, hipStream_t stream, bool launch);

} // namespace tenmo
#endif
