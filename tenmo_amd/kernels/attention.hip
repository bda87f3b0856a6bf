// Entry points of attention (include/tenmo_hip_transformer.h): checks, and which kernels a call takes.
#include "attention.hpp"

namespace tenmo {
namespace {

// Launches hold 2^32 threads, and indexes of rows 31 bits; the operands' own offsets are 64 bits.
int attn_shape(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim, const char* who, AttnShape* s) {
    if (batch < 0 || queries < 0 || keys < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads)
        return refuse(TENMO_ERR_INVALID_SHAPE, "%s: %lld query heads for %lld key heads: a multiple of them is needed", who, (long long)heads, (long long)kv_heads);
    if (dim < 1 || dim > 128) return refuse(TENMO_ERR_UNSUPPORTED, "%s: head size %lld, 1 to 128 are supported", who, (long long)dim);
    const int64_t sequences = 1 << 20, rows = 1 << 25, keys_most = 1 << 27; // (each below what makes the next product overflow)
    if (batch > sequences || heads > sequences || batch * heads > sequences || queries > rows || keys > keys_most || batch * heads * queries > rows || batch * kv_heads * keys > keys_most)
        return refuse(TENMO_ERR_UNSUPPORTED, "%s: more than 2^20 heads of sequences, 2^25 rows of queries or 2^27 of keys", who);
    s->batch = (int)batch; s->queries = (int)queries; s->keys = (int)keys; s->heads = (int)heads; s->kv_heads = (int)kv_heads; s->dim = (int)dim;
    s->group = (int)(heads / kv_heads);
    return 0;
}

AttnOperand operand_of(const tenmo_view* v) {
    if (!v) return AttnOperand{nullptr, 0, 0, 0, 0};
    return AttnOperand{v->data ? const_cast<float*>(v->data) + v->offset : nullptr, v->strides[0], v->strides[1], v->strides[2], v->strides[3]};
}

int check_qkv(const tenmo_view* Q, const tenmo_view* K, const tenmo_view* V, float scale, const char* who, AttnShape* s) {
    if (int rc = check_operand(Q, 4, 4, who, "Q")) return rc;
    if (int rc = check_operand(K, 4, 4, who, "K")) return rc;
    if (int rc = check_operand(V, 4, 4, who, "V")) return rc;
    if (K->shape[0] != Q->shape[0] || K->shape[3] != Q->shape[3])
        return refuse(TENMO_ERR_INVALID_SHAPE, "%s: batch and head size of Q (%lld, %lld) and K (%lld, %lld) differ", who, (long long)Q->shape[0], (long long)Q->shape[3],
                      (long long)K->shape[0], (long long)K->shape[3]);
    for (int d = 0; d < 4; ++d)
        if (V->shape[d] != K->shape[d])
            return refuse(TENMO_ERR_INVALID_SHAPE, "%s: axis %d of V has %lld elements, of K %lld", who, d, (long long)V->shape[d], (long long)K->shape[d]);
    if (!(scale - scale == 0.f)) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: scale is not finite", who);
    if (int rc = attn_shape(Q->shape[0], Q->shape[1], K->shape[1], Q->shape[2], K->shape[2], Q->shape[3], who, s)) return rc;
    s->scale = scale;
    return 0;
}

int check_gradient(const tenmo_view* g, const tenmo_view* of, const char* who, const char* what) {
    if (!g) return 0;
    if (int rc = check_operand(g, 4, 4, who, what)) return rc;
    for (int d = 0; d < 4; ++d) {
        if (g->shape[d] != of->shape[d])
            return refuse(TENMO_ERR_INVALID_SHAPE, "%s: axis %d of %s has %lld elements, %lld needed", who, d, what, (long long)g->shape[d], (long long)of->shape[d]);
        if (g->shape[d] > 1 && g->strides[d] == 0 && elements(g) > 0) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: %s has a stride of 0: its elements share a place", who, what);
    }
    return 0;
}

__global__ __launch_bounds__(256) void attn_zero_kernel(AttnOperand g, int64_t n, int s, int h, int d) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / d, t = r / h;
        g.p[t / s * g.b + t % s * g.s + r % h * g.h + i % d * g.d] = 0.f;
    }
}

// Rows or tiles.  Rows cost by pairs of a query and a key, tiles begin with two launches and one more pass over the operands: by these sums, fitted to 264 launches of
// D = 32, 64, 128 with 2 to 512 queries, 64 to 8192 keys and 8 to 512 heads.  No choice costs more than 1.4 of the other there, and 1 % in the mean; at [1, 8 x 64, 64 keys] rows take
// 13 us and tiles 20, at [32,16 x 64, 256 keys] 382 and 74.
double padded(int dim) { return (dim + 31) / 32 * 32; }
double pair_values(const AttnShape& s) { return (double)s.batch * s.heads * s.queries * s.keys * padded(s.dim); }
bool forward_by_rows(const AttnShape& s) {
    const double operands = (double)s.batch * padded(s.dim) * ((double)s.heads * s.queries + 2.0 * s.kv_heads * s.keys);
    return pair_values(s) <= 60e6 + 15.0 * operands;
}
// Backward, where a wavefront takes the keys of its row one after the other, two a slot at a time: that chain counts besides, 1024 of them at most.  No choice costs more than 1.34 of the
// other, and 1 % in the mean; [1, 8 x 64]: 128 queries and keys take 18 us by rows and 31 by tiles, 512 of both 83 and 49.
bool backward_by_rows(const AttnShape& s) {
    const double operands = 2.0 * s.batch * padded(s.dim) * ((double)s.heads * s.queries + (double)s.kv_heads * s.keys);
    const bool fits = (int64_t)s.batch * s.kv_heads * s.keys < 1 << 24; // a launch: half as many workgroups at the most
    return fits && s.queries <= 1024 && s.keys <= 1024 && pair_values(s) + 800.0 * padded(s.dim) * s.keys <= 60e6 + 2.0 * operands;
}

// Tiles hold 2^24 workgroups a launch, and a part of each query head's share of dK and dV.
int backward_fits(const AttnShape& s, const char* who) {
    if (s.group > 1 && !backward_by_rows(s) && (int64_t)s.batch * s.heads * s.keys > 1 << 28)
        return refuse(TENMO_ERR_UNSUPPORTED, "%s: more than 2^28 rows of keys over all query heads", who);
    return 0;
}

void forward_plan(const AttnShape& s, const AttnOperand& q, const AttnOperand& k, const AttnOperand& v, float* out, float* lse, Workspace& ws, const LibraryState& lib, bool launch) {
    if (forward_by_rows(s)) attn_rows_forward(s, q, k, v, out, lse, ws, lib.cus, lib.stream, launch);
    else attn_tiles_forward(s, q, k, v, out, lse, ws, lib.cus, lib.stream, launch);
}

void backward_plan(const AttnBackward& b, Workspace& ws, const LibraryState& lib, bool launch) {
    if (!backward_by_rows(b.s)) attn_tiles_backward(b, ws, lib.cus, lib.stream, launch);
    else if (launch) attn_rows_backward(b, lib.stream);
}

} // namespace
} // namespace tenmo

using namespace tenmo;

extern "C" {

int64_t tenmo_hip_attention_forward_workspace_bytes(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    AttnShape s{};
    LibraryState lib{};
    if (int rc = attn_shape(batch, queries, keys, heads, kv_heads, dim, "tenmo_hip_attention_forward_workspace_bytes", &s)) return rc;
    if (int rc = library_state(&lib)) return rc;
    Workspace ws(nullptr, 0);
    if (batch > 0 && queries > 0) forward_plan(s, AttnOperand{}, AttnOperand{}, AttnOperand{}, nullptr, nullptr, ws, lib, false);
    return ws.used();
}

int tenmo_hip_attention_forward_f32(const tenmo_view* Q, const tenmo_view* K, const tenmo_view* V, float scale, int32_t causal,
                                    const int32_t* key_lengths, const int32_t* query_starts, float* out, float* lse,
                                    void* workspace, int64_t workspace_bytes, int32_t sync) {
    const char* who = "tenmo_hip_attention_forward_f32";
    AttnShape s{};
    if (int rc = check_qkv(Q, K, V, scale, who, &s)) return rc;
    const bool none = s.batch == 0 || s.queries == 0;
    if (!out && !none) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: null out", who);
    Call call(who);
    if (int rc = call.begin()) return rc;
    if (none) return 0;
    s.causal = causal != 0; s.key_lengths = key_lengths; s.query_starts = query_starts;
    Workspace ws(workspace, workspace_bytes);
    forward_plan(s, operand_of(Q), operand_of(K), operand_of(V), out, lse, ws, call.state, false);
    if (int rc = ws.check(who)) return rc;
    ws = Workspace(workspace, workspace_bytes);
    forward_plan(s, operand_of(Q), operand_of(K), operand_of(V), out, lse, ws, call.state, true);
    return call.finish(sync);
}

int64_t tenmo_hip_attention_backward_workspace_bytes(int64_t batch, int64_t queries, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
    AttnBackward b{};
    LibraryState lib{};
    if (int rc = attn_shape(batch, queries, keys, heads, kv_heads, dim, "tenmo_hip_attention_backward_workspace_bytes", &b.s)) return rc;
    if (int rc = backward_fits(b.s, "tenmo_hip_attention_backward_workspace_bytes")) return rc;
    if (int rc = library_state(&lib)) return rc;
    Workspace ws(nullptr, 0);
    if (batch > 0 && queries > 0 && keys > 0) backward_plan(b, ws, lib, false);
    return ws.used();
}

int tenmo_hip_attention_backward_f32(const tenmo_view* Q, const tenmo_view* K, const tenmo_view* V, float scale, int32_t causal,
                                     const int32_t* key_lengths, const int32_t* query_starts, const float* out, const float* lse,
                                     const float* dOut, const tenmo_view* grad_Q, const tenmo_view* grad_K, const tenmo_view* grad_V,
                                     int32_t accumulate, void* workspace, int64_t workspace_bytes, int32_t sync) {
    const char* who = "tenmo_hip_attention_backward_f32";
    AttnBackward b{};
    if (int rc = check_qkv(Q, K, V, scale, who, &b.s)) return rc;
    if (int rc = check_gradient(grad_Q, Q, who, "grad_Q")) return rc;
    if (int rc = check_gradient(grad_K, K, who, "grad_K")) return rc;
    if (int rc = check_gradient(grad_V, V, who, "grad_V")) return rc;
    const AttnShape& s = b.s;
    if (int rc = backward_fits(s, who)) return rc;
    if (s.batch > 0 && s.queries > 0 && s.keys > 0 && (!out || !lse || !dOut)) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: null out, lse or dOut", who);
    Call call(who);
    if (int rc = call.begin()) return rc;
    if (s.batch == 0 || (!grad_Q && !grad_K && !grad_V)) return 0;
    b.q = operand_of(Q); b.k = operand_of(K); b.v = operand_of(V);
    b.grad_q = operand_of(grad_Q); b.grad_k = operand_of(grad_K); b.grad_v = operand_of(grad_V);
    if (s.queries == 0 || s.keys == 0) { // nothing attends to anything: the gradients of what is there are zero
        if (accumulate) return 0;
        auto zero = [&](const AttnOperand& g, int64_t n, int h) {
            const int64_t all = (int64_t)s.batch * n * h * s.dim;
            if (g.p && all) hipLaunchKernelGGL(attn_zero_kernel, dim3((unsigned)(all < 256 * 1024 ? (all + 255) / 256 : 1024)), dim3(256), 0, call.state.stream, g, all, (int)n, h, s.dim);
        };
        zero(b.grad_q, s.queries, s.heads);
        zero(b.grad_k, s.keys, s.kv_heads);
        zero(b.grad_v, s.keys, s.kv_heads);
        return call.finish(sync);
    }
    b.s.causal = causal != 0; b.s.key_lengths = key_lengths; b.s.query_starts = query_starts;
    b.out = out; b.lse = lse; b.dout = dOut; b.accumulate = accumulate ? 1 : 0;
    Workspace ws(workspace, workspace_bytes);
    backward_plan(b, ws, call.state, false);
    if (int rc = ws.check(who)) return rc;
    ws = Workspace(workspace, workspace_bytes);
    backward_plan(b, ws, call.state, true);
    return call.finish(sync);
}

} // extern "C"
