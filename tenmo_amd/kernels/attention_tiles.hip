// Attention for many query rows, forward and backward, on the fp16 matrix units (the split products of split_gemm.hpp).
//
// Forward, a wavefront for 32 queries, 32 keys at a time:
//   S^T = K Q^T (keys x queries), p = 2^(S c - m + 7) with c = scale log2(e), O^T += V^T P^T, l += sum p.
// (Backward, a wavefront works on the up to three tiles of its workgroup that are beyond its own rows as on any other: leaving them out made the
// compiler copy its sums, 250 instructions a tile.)
// S^T comes out of the matrix units with a query in each lane (twice: the halves hold the keys 8 a + 0..3 and 8 a + 4..7), so the softmax needs one
// exchange between lanes, and its registers are the operand of the second product as they are: the order in which that product takes the keys is free, and V is
// fetched in the same one.  The running maximum m is renewed when a score passes it by 2^8 (p and the sums keep to the range of their types below that).
//
// Backward, the probabilities again, without atomics and so without an order:
//   keys:    a wavefront for 32 keys of a query head, over the queries that see them: S = Q K^T, dP = dO V^T,
//            P = 2^(S c - lse), dS = P (dP - delta); dV^T += dO^T P, dK^T += Q^T dS.
//   queries: a wavefront for 32 queries, over their keys: S^T, dP^T, dS^T; dQ^T += K^T dS^T.
// Seven products for the five that one pass with atomics would need.
//
// The operands that are read in tiles are brought into split form first, head by head, rows padded to 128 and D to DP = 32, 64, 96 or 128 with zeros; rows that no allowed pair touches are
// zeros too, whatever the operand holds there.
//   * forward, K and V in one launch: 64 rows have a scale of their own (one read, where a scale of the whole head takes a launch before: [8,1024,12,64] 84 -> 71 us, [4,777,16,80] 73 -> 59).
//     A wavefront's own rows of q are split as they are read, with a scale of their own each.
//   * backward, all four in two launches: the largest magnitudes (of the rows that count), then the halves, with one scale a head for Q, K and V and one a row for dO.
//
// What a row of a gradient is summed from is held to the row's own sizes, however small they are against the head's (with one scale a head, keys of a weight of e^-18 got dK to 0.1 of itself,
// and rows of dQ where dO is 2^-20 of the head's largest to 0.05):
//   * a row of dO that is small against the head's largest has a scale a_i of its own, and P is taken times A / a_i (A: the head's scale): P dO is the same, and what the row adds is small in P
//     instead (zeros: nothing).  The factor goes into the row's lse.
//   * P and dS have a scale for each row of the result, which is a lane: a power of two that brings the largest so far into 2^10 .. 2^15, renewed, with the sums, when one passes it.
//     Since it is known only when a tile is done, it costs a maximum of the tile's 16 values and a branch (the kernel at [8,1024,12,64] 187 us with and without, at [1,8192,16/4,128] 2967 and
//     2960; with 2^12 in place of 2^10 scales are renewed more often: 194 and 3150, and with sums moved by the compiler, see scale_sums, 200 and 3670).
//
// LDS tile: 32 rows of DP / 4 chunks of 16 bytes, chunk c = 2 * (d / 8) + kind at slot c ^ swizzle(row); read by rows (16 bytes a lane: 16 rows in 16 different slots of the
// banks) and by columns (the transposing read: 4 rows x 4 chunks in 16 different slots).
#include "attention.hpp"
#include "split_gemm.hpp"

#include <algorithm>

namespace tenmo {
namespace {

constexpr int kRowPad = 128;        // rows of a head are padded to the rows of a workgroup
constexpr int kHeadParts = 32;      // partial maxima of a head
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kPBits = 7.f;       // p is held as p 2^7
constexpr float kRenew = 8.f;

__host__ __device__ constexpr int row_pad(int n) { return (n + kRowPad - 1) / kRowPad * kRowPad; }

enum { kK, kV, kQ, kDO }; // forward the first two are split beforehand, backward all of them

// Of a row of queries, backward, with a_i the scale of the row of dO and A the head's: lse log2(e) + log2(a_i / A) (+inf where there is no lse: no probability), dO . O times a_i / A, A / a_i, dO . O
enum { kLseUp, kDeltaUp, kDown, kDelta, kStats };
__device__ __forceinline__ int64_t stat_at(int64_t row, int which) { return (row >> 5) * (32 * kStats) + which * 32 + (row & 31); }

struct TileArgs {
    AttnShape s;
    AttnOperand src[4];
    int parts;          // runs of a head's rows in the first launch
    float* split[4];    // [batch][heads][rows padded][DP]
    f32x4* seen[4];     // [batch * heads][parts]: of a run of rows, the largest finite magnitude, the largest norm of a row, the smallest largest magnitude of a row
                        // that is not zero, and 1 if there is a value that is not finite
    f32x4* head[4];     // [batch * heads]: scale, largest norm of a row, 1 if the halves do not hold this head (backward)
    const float *out, *lse;
    float* stats;        // backward, [batch][heads][queries padded / 32][kStats][32] (and 4 tiles behind the last)
    // forward
    float* scale[2];     // [batch * heads][blocks of 64 rows]: 1 / the scale of K, the scale of V or 0 where there are zeros alone; `seen` is of these blocks too
    float *to, *to_lse, *part;
    int splits;
    // backward
    AttnOperand grad_q, grad_k, grad_v;
    int accumulate;
    int query_runs, key_runs;       // into which the queries of a block of keys, and the keys of a block of queries, are cut
    float *part_k, *part_v, *part_q; // [runs][batch][heads][rows][dim]: the parts of each run and query head, where there is more than one
};

// first query row with a key, and the number of keys that some query may use
__device__ __forceinline__ int first_query(const AttnShape& s, int length, int start) { return length == 0 ? s.queries : start < 0 ? -start : 0; }
__device__ __forceinline__ int used_keys(const AttnShape& s, int length, int start) { return attn_limit(length, start, s.queries - 1); }

struct HeadJob {
    int job, heads, bh, b, h, rows, pad;
    int lo, hi; // the rows that count
    AttnOperand src;
    float* split;
    f32x4 *seen, *head;
};
// (the operand is picked by comparisons: an index into the arguments that is not known to the compiler would put them into scratch memory)
__device__ __forceinline__ HeadJob head_job(const TileArgs& a, int y) {
    HeadJob j;
    const int q = a.s.batch * a.s.heads, k = a.s.batch * a.s.kv_heads;
    j.job = y < k ? kK : y < 2 * k ? kV : y < 2 * k + q ? kQ : kDO;
    const bool key = j.job == kK || j.job == kV;
    j.bh = j.job == kK ? y : j.job == kV ? y - k : j.job == kQ ? y - 2 * k : y - 2 * k - q;
    j.heads = key ? a.s.kv_heads : a.s.heads;
    j.b = j.bh / j.heads;
    j.h = j.bh - j.b * j.heads;
    j.rows = key ? a.s.keys : a.s.queries;
    j.pad = row_pad(j.rows);
    const int length = attn_length(a.s, j.b), start = attn_start(a.s, j.b);
    j.lo = key ? 0 : first_query(a.s, length, start);
    j.hi = key ? used_keys(a.s, length, start) : a.s.queries;
#define TENMO_PICK(x) (j.job == kQ ? a.x[kQ] : j.job == kK ? a.x[kK] : j.job == kV ? a.x[kV] : a.x[kDO])
    j.src.p = TENMO_PICK(src).p;
    j.src.b = TENMO_PICK(src).b;
    j.src.s = TENMO_PICK(src).s;
    j.src.h = TENMO_PICK(src).h;
    j.src.d = TENMO_PICK(src).d;
    j.split = TENMO_PICK(split);
    j.seen = TENMO_PICK(seen);
    j.head = TENMO_PICK(head);
#undef TENMO_PICK
    return j;
}

// of a power of two
__device__ __forceinline__ float power_inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

// What a run of a head's rows holds, and each row's lse, delta and largest magnitude of dO: L lanes a row, U rows in flight
template <int L>
__global__ __launch_bounds__(256) void attn_amax_kernel(const TileArgs a) {
    constexpr int SLOTS = 64 / L, U = 4;
    __shared__ f32x4 seen_of[4];
    const int run = blockIdx.x % a.parts;
    const HeadJob j = head_job(a, blockIdx.x / a.parts);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = lane % L, D = a.s.dim;
    const float* p = j.src.p + j.b * j.src.b + j.h * j.src.h;
    const int all = j.job == kDO ? j.pad : j.rows, per = (all + a.parts - 1) / a.parts;
    const int first = run * per, last = first + per < all ? first + per : all;
    float top = 0.f, norm = 0.f, least = __builtin_inff();
    bool wrong = false;
    for (int r0 = first + wave * SLOTS + lane / L; __any(r0 < last); r0 += 4 * SLOTS * U) {
        f32x4 x[U], o[U];
        // (a row that does not count is read as one that does, or as the first)
        auto row_at = [&](int u) { const int r = r0 + 4 * SLOTS * u; return r >= j.lo && r < j.hi ? r : j.lo < j.hi ? j.lo : 0; };
        attn_with_kind(attn_kind(j.src.d, D), [&](auto kind) {
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = attn_load4<kind.value>(p + row_at(u) * j.src.s, j.src.d, part, D);
        });
        if (j.job == kDO)
            attn_with_kind(attn_kind(1, D), [&](auto kind) {
#pragma unroll
                for (int u = 0; u < U; ++u) o[u] = attn_load4<kind.value>(a.out + (((int64_t)j.b * a.s.queries + row_at(u)) * a.s.heads + j.h) * D, 1, part, D);
            });
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + 4 * SLOTS * u;
            const bool in = r < last && r >= j.lo && r < j.hi;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][e] = in ? x[u][e] : 0.f;
            float mine = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                mine = fmaxf(mine, __uint_as_float(finite_magnitude(x[u][e])));
                wrong |= !(x[u][e] - x[u][e] == 0.f);
            }
            mine = lanes_max<L>(mine);
            top = fmaxf(top, mine);
            if (mine > 0.f) least = fminf(least, mine);
            const float sq = lanes_sum<L>(dot4(x[u], x[u]));
            // (a square out of range: the largest magnitude times sqrt(D) instead)
            norm = fmaxf(norm, sq < 1e37f && sq > 1e-30f ? sqrtf(sq) : fminf(mine * sqrtf((float)D), 1e38f));
            if (j.job == kDO) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[u][e] = in ? o[u][e] : 0.f;
                const float delta = lanes_sum<L>(dot4(x[u], o[u]));
                if (part == 0 && r < last) {
                    const int64_t row = (int64_t)j.bh * j.pad + r;
                    a.stats[stat_at(row, kLseUp)] = in ? a.lse[(int64_t)j.bh * a.s.queries + r] * kLog2e : __builtin_inff();
                    a.stats[stat_at(row, kDown)] = mine; // the next launch makes a scale of it
                    a.stats[stat_at(row, kDelta)] = in ? delta : 0.f;
                }
            }
        }
    }
    const f32x4 mine{wave_max(top), wave_max(norm), -wave_max(-least), __any(wrong) ? 1.f : 0.f};
    if (lane == 0) seen_of[wave] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        f32x4 s = seen_of[0];
        for (int w = 1; w < 4; ++w) s = f32x4{fmaxf(s[0], seen_of[w][0]), fmaxf(s[1], seen_of[w][1]), fminf(s[2], seen_of[w][2]), fmaxf(s[3], seen_of[w][3])};
        j.seen[(int64_t)j.bh * a.parts + run] = s;
    }
}

// The halves of 64 rows, 8 values a thread; the first workgroup of a head leaves what the products need to know of it.
// The halves hold a value to 2^-22 of itself and 2^-40 of the largest that has the same scale.  With one scale a head that is taken while no row that is not zero is smaller than 2^-16 of the
// largest: 2^-24 of each row's own.  Rows of dout lie further apart (gradients of single positions do) and have a scale of their own.
template <int DP>
__global__ __launch_bounds__(256) void attn_split_kernel(const TileArgs a) {
    constexpr int GROUPS = DP / 8, ROWS = 64, N = ROWS * GROUPS / 256;
    // the heads of K and V first
    const uint32_t key_blocks = row_pad(a.s.keys) / ROWS, query_blocks = row_pad(a.s.queries) / ROWS, key_heads = 2 * a.s.batch * a.s.kv_heads;
    const bool key = blockIdx.x < key_heads * key_blocks;
    const uint32_t id = key ? blockIdx.x : blockIdx.x - key_heads * key_blocks, blocks = key ? key_blocks : query_blocks;
    const int block = id % blocks;
    const HeadJob j = head_job(a, (key ? 0 : key_heads) + id / blocks);
    const int lane = threadIdx.x & 63;
    f32x4 s{0.f, 0.f, __builtin_inff(), 0.f};
    if (lane < a.parts) s = j.seen[(int64_t)j.bh * a.parts + lane];
    const float top = wave_max(s[0]), scale = split_scale(__float_as_uint(top));
    if (block == 0) {
        const float norm = wave_max(s[1]), least = -wave_max(-s[2]), wrong = wave_max(s[3]);
        if (threadIdx.x == 0) j.head[j.bh] = f32x4{scale, norm, wrong > 0.f || (j.job != kDO && top * 0x1p-16f > least) ? 1.f : 0.f, 0.f};
    }
    const float* p = j.src.p + j.b * j.src.b + j.h * j.src.h;
    f32x4 v[N][2];
    attn_with_kind(attn_kind(j.src.d, a.s.dim), [&](auto kind) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = threadIdx.x + 256 * i, r = block * ROWS + x / GROUPS, at = r >= j.lo && r < j.hi ? r : j.lo < j.hi ? j.lo : 0;
#pragma unroll
            for (int u = 0; u < 2; ++u) v[i][u] = attn_load4<kind.value>(p + at * j.src.s, j.src.d, x % GROUPS * 2 + u, a.s.dim);
        }
    });
    float scales[N], ups[N]; // ups: scales over the head's
#pragma unroll
    for (int i = 0; i < N; ++i) scales[i] = scale, ups[i] = 1.f;
    if (j.job == kDO) { // (in the whole workgroup)
#pragma unroll
        for (int i = 0; i < N; ++i) { // (at most 2^120 times the head's, so that the quotient of the two is a float; 2^-12 of the largest is held to 2^-28 by the head's)
            const float mine = a.stats[stat_at((int64_t)j.bh * j.pad + block * ROWS + (threadIdx.x + 256 * i) / GROUPS, kDown)];
            if (mine > 0.f && mine < top * 0x1p-12f) scales[i] = fminf(split_scale(__float_as_uint(mine)), scale * 0x1p120f), ups[i] = scales[i] * power_inverse(scale);
            if (mine == 0.f) ups[i] = 0x1p120f; // a row of zeros takes the smallest P: it leaves the scale that the others' have as it is
        }
        __syncthreads(); // each row's magnitude is read by all of its threads before one of them writes in its place
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = threadIdx.x + 256 * i;
            if (x % GROUPS) continue;
            const int64_t row = (int64_t)j.bh * j.pad + block * ROWS + x / GROUPS;
            const float up = ups[i];
            a.stats[stat_at(row, kLseUp)] += (float)((int)(__float_as_uint(up) >> 23) - 127);
            a.stats[stat_at(row, kDeltaUp)] = a.stats[stat_at(row, kDelta)] * up;
            a.stats[stat_at(row, kDown)] = power_inverse(up);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int x = threadIdx.x + 256 * i, r = block * ROWS + x / GROUPS;
        const bool in = r >= j.lo && r < j.hi;
        f16x8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 hi16, lo16;
            split_value(in ? v[i][e >> 2][e & 3] * scales[i] : 0.f, hi16, lo16);
            h[e] = hi16;
            l[e] = lo16;
        }
        float* to = j.split + ((int64_t)j.bh * j.pad + r) * DP + x % GROUPS * 8;
        *(f16x8*)to = h;
        *(f16x8*)(to + 4) = l;
    }
}

__device__ __forceinline__ float lane_value(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }

// Forward, K and V in one launch: a workgroup reads 64 rows, 4 values a lane and L lanes a row, and gives them a scale of their own.
template <int DP, int L>
__global__ __launch_bounds__(256) void attn_prepare_kernel(const TileArgs a) {
    constexpr int SLOTS = 64 / L, U = L / 4, ROWS = 64; // U * 4 * SLOTS rows
    __shared__ f32x4 seen_of[4];
    const int blocks = row_pad(a.s.keys) / ROWS, block = blockIdx.x % blocks;
    const HeadJob j = head_job(a, blockIdx.x / blocks);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = lane % L, D = a.s.dim;
    const float* p = j.src.p + j.b * j.src.b + j.h * j.src.h;
    auto row_of = [&](int u) { return block * ROWS + (u * 4 + wave) * SLOTS + lane / L; };
    f32x4 x[U];
    attn_with_kind(attn_kind(j.src.d, D), [&](auto kind) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = attn_load4<kind.value>(p + (row_of(u) < j.hi ? row_of(u) : 0) * j.src.s, j.src.d, part, D); // (a row that does not count is read as the first)
    });
    float top = 0.f, least = __builtin_inff();
    bool wrong = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool in = row_of(u) < j.hi;
        float mine = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[u][e] = in ? x[u][e] : 0.f;
            mine = fmaxf(mine, __uint_as_float(finite_magnitude(x[u][e])));
            wrong |= !(x[u][e] - x[u][e] == 0.f);
        }
        mine = lanes_max<L>(mine);
        top = fmaxf(top, mine);
        if (mine > 0.f) least = fminf(least, mine);
    }
    const f32x4 mine{wave_max(top), 0.f, -wave_max(-least), __any(wrong) ? 1.f : 0.f};
    if (lane == 0) seen_of[wave] = mine;
    __syncthreads();
    f32x4 s = seen_of[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) s = f32x4{fmaxf(s[0], seen_of[w][0]), 0.f, fminf(s[2], seen_of[w][2]), fmaxf(s[3], seen_of[w][3])};
    const float scale = split_scale(__float_as_uint(s[0]));
    if (threadIdx.x == 0) {
        j.seen[(int64_t)j.bh * blocks + block] = s;
        (j.job == kK ? a.scale[kK] : a.scale[kV])[(int64_t)j.bh * blocks + block] = j.job == kK ? power_inverse(scale) : s[0] > 0.f ? scale : 0.f;
    }
    if (4 * part >= DP) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        f16x4 h, l;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            _Float16 hi16, lo16;
            split_value(x[u][e] * scale, hi16, lo16);
            h[e] = hi16;
            l[e] = lo16;
        }
        // 8 h, then 8 l: two lanes have four of each
        float* to = j.split + ((int64_t)j.bh * j.pad + row_of(u)) * DP + part / 2 * 8 + part % 2 * 2;
        *(f16x4*)to = h;
        *(f16x4*)(to + 4) = l;
    }
}

// Whether the halves do not hold K or V of this head: from what its blocks hold, in every lane
__device__ __forceinline__ bool keys_beyond(const TileArgs& a, int bk) {
    const int blocks = row_pad(a.s.keys) / 64, lane = threadIdx.x & 63;
    bool bad = false;
#pragma unroll
    for (int job = 0; job < 2; ++job) {
        float top = 0.f, least = __builtin_inff(), wrong = 0.f;
        for (int i = lane; i < blocks; i += 64) {
            const f32x4 s = a.seen[job][(int64_t)bk * blocks + i];
            top = fmaxf(top, s[0]);
            least = fminf(least, s[2]);
            wrong = fmaxf(wrong, s[3]);
        }
        bad |= __any(wrong > 0.f) || wave_max(top) * 0x1p-16f > -wave_max(-least);
    }
    return bad;
}

// Heads beyond the halves are worked on row by row in fp32, where nothing that is not allowed can leave a trace: those with keys or values that are not finite, or of sizes too far apart;
// and backward the same of q, dout that is not finite, and scores above 2^16 (|q| |k| scale; with one scale for all rows of q their error would pass 2^-24).
__device__ __forceinline__ bool beyond(const TileArgs& a, f32x4 q, f32x4 k, f32x4 v) { return q[2] + k[2] + v[2] > 0.f || !(q[1] * k[1] * fabsf(a.s.scale) < 65536.f); }

__device__ __forceinline__ void store_part(float* to, int d, int D, f32x4 x) {
    if (d + 3 < D) *(f32x4_u*)(to + d) = x;
    else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < D) to[d + e] = x[e];
}

// ---- heads beyond the halves: a wavefront a row, or 64 / L keys ------------------------------------------------------------------------

__device__ __forceinline__ f32x4 slow_load(const AttnOperand& o, int b, int64_t s, int h, int part, int D) {
    return attn_load4<kLoadAny>(o.p + b * o.b + s * o.s + h * o.h, o.d, part, D);
}

// a row's sum of p v (this lane's four values), its maximum and sum over the keys lo .. hi - 1
template <int L>
__device__ __forceinline__ f32x4 slow_forward(const TileArgs& a, int b, int h, int i, int lo, int hi, float& m, float& l) {
    constexpr int SLOTS = 64 / L;
    const int lane = threadIdx.x & 63, part = lane % L, D = a.s.dim, hk = h / a.s.group;
    const f32x4 q = slow_load(a.src[kQ], b, i, h, part, D) * a.s.scale;
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    m = kNone;
    l = 0.f;
    for (int j = lo + lane / L; __any(j < hi); j += SLOTS) {
        const int jr = j < hi ? j : hi - 1;
        const f32x4 k = slow_load(a.src[kK], b, jr, hk, part, D), v = slow_load(a.src[kV], b, jr, hk, part, D);
        const float x = lanes_sum<L>(dot4(q, k));
        if (j < hi) {
            const float top = fmaxf(m, x), keep = below(m, top), p = below(x, top);
            l = l * keep + p;
            o = o * keep + p * v;
            m = top;
        }
    }
#pragma unroll
    for (int d = L; d < 64; d <<= 1) {
        const float om = __shfl_xor(m, d, 64), top = fmaxf(m, om), keep = below(m, top), okeep = below(om, top);
        l = l * keep + __shfl_xor(l, d, 64) * okeep;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * keep + __shfl_xor(o[e], d, 64) * okeep;
        m = top;
    }
    return o;
}

// a row of dQ, without its factor scale
template <int L>
__device__ __forceinline__ f32x4 slow_dq(const TileArgs& a, int b, int h, int i, int lo, int limit, float lse, float delta) { // from the keys lo .. limit - 1
    constexpr int SLOTS = 64 / L;
    const int lane = threadIdx.x & 63, part = lane % L, D = a.s.dim, hk = h / a.s.group;
    const f32x4 q = slow_load(a.src[kQ], b, i, h, part, D) * a.s.scale, g = slow_load(a.src[kDO], b, i, h, part, D);
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int j = lo + lane / L; __any(j < limit); j += SLOTS) {
        const int jr = j < limit ? j : limit - 1;
        const f32x4 k = slow_load(a.src[kK], b, jr, hk, part, D), v = slow_load(a.src[kV], b, jr, hk, part, D);
        const float x = lanes_sum<L>(dot4(q, k)), dp = lanes_sum<L>(dot4(g, v));
        if (j < limit) acc += __expf(x - lse) * (dp - delta) * k;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = L; d < 64; d <<= 1) acc[e] += __shfl_xor(acc[e], d, 64);
    return acc;
}

// dK (without its factor scale) and dV of a key of this slot's, from the queries lo .. hi - 1 of head h
template <int L>
__device__ __forceinline__ void slow_dkv(const TileArgs& a, int b, int h, int j, int length, int start, int lo, int hi, f32x4& dk, f32x4& dv) {
    const int part = (threadIdx.x & 63) % L, D = a.s.dim, hk = h / a.s.group, jr = j < a.s.keys ? j : a.s.keys - 1;
    const int64_t bh = (int64_t)b * a.s.heads + h;
    const f32x4 k = slow_load(a.src[kK], b, jr, hk, part, D), v = slow_load(a.src[kV], b, jr, hk, part, D);
    dk = dv = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = lo; i < hi; ++i) {
        const int limit = attn_limit(length, start, i);
        if (!__any(j < limit)) continue;
        const f32x4 q = slow_load(a.src[kQ], b, i, h, part, D), g = slow_load(a.src[kDO], b, i, h, part, D);
        const float x = lanes_sum<L>(dot4(q, k)) * a.s.scale, dp = lanes_sum<L>(dot4(g, v));
        if (j < limit) {
            const float p = __expf(x - a.lse[bh * a.s.queries + i]);
            dv += p * g;
            dk += p * (dp - a.stats[stat_at(bh * row_pad(a.s.queries) + i, kDelta)]) * q;
        }
    }
}

// ---- tiles in LDS ------------------------------------------------------------------------------------------------------------------

template <int DP>
struct Tile {
    static constexpr int CH = DP / 4, KD = DP / 16, ND = DP / 32, BYTES = 32 * CH * 16, BLOCKS = BYTES / 1024;
    static constexpr bool WIDE = DP % 64 == 0;
    static constexpr int LANES = DP <= 32 ? 8 : DP <= 64 ? 16 : 32; // of a row in fp32, four values each

    static __device__ __forceinline__ int swizzle(int row) { return WIDE ? (row & 1) | ((row >> 1) & 6) | ((row & 2) << 2) : (row >> 1) & 7; }

    // this lane's byte offsets for the 1 KiB blocks wave, wave + 4, .. of N tiles that lie one behind the other
    template <int N>
    static __device__ __forceinline__ void offsets(uint32_t (&off)[N * BLOCKS / 4], int wave, int lane) {
#pragma unroll
        for (int i = 0; i < N * BLOCKS / 4; ++i) {
            const int x = (i * 4 + wave) % BLOCKS * 64 + lane, row = x / CH, slot = x % CH;
            off[i] = (uint32_t)(row * CH + (slot ^ swizzle(row))) * 16u;
        }
    }
    // N tiles from src[0 ..] (the same rows of N operands) into LDS
    template <int N>
    static __device__ __forceinline__ void load(float* lds, uint32_t at, const float* const (&src)[N], const uint32_t (&off)[N * BLOCKS / 4], int wave) {
#pragma unroll
        for (int i = 0; i < N * BLOCKS / 4; ++i) {
            const int block = i * 4 + wave; // blocks of a tile come in fours: the tile does not depend on the wavefront
            direct_load_16B(lds, at + (uint32_t)block * 1024u, off[i], src[i * 4 / BLOCKS]);
        }
    }
    // row operand: lane % 32 is the row, lane / 32 the half of 16 values of d
    static __device__ __forceinline__ uint32_t row_offset(int lane, int kind) {
        const int r = lane & 31;
        return (uint32_t)(r * CH + ((2 * (lane >> 5) + kind) ^ swizzle(r))) * 16u;
    }
    static __device__ __forceinline__ f16x8 row_read(const char* tile, uint32_t off, int ks) {
        constexpr int XM = WIDE ? 3 : 1;
        return *(const f16x8*)(tile + (off ^ ((ks & XM) * 64)) + (ks & ~XM) * 64);
    }
    // column operand: lane % 32 is the value of d (of 32), the 8 values rows 16 t + 4 (lane / 32) + {0..3, 8..11}
    static __device__ __forceinline__ uint32_t column_offset(int lane, int kind) {
        const int p = lane & 15, sub = (lane >> 4) & 1, row = 4 * (lane >> 5) + (p >> 2);
        return (uint32_t)(row * CH + ((4 * sub + 2 * ((p & 3) >> 1) + kind) ^ swizzle(row))) * 16u + 8u * (p & 1);
    }
    static __device__ __forceinline__ f16x8 column_read(const char* tile, uint32_t off, int t, int db) {
        typedef __attribute__((address_space(3))) i16x4* lds_p;
        union { i16x4 s[2]; f16x8 v; } x;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t at = WIDE ? (off ^ (u * 64) ^ ((db & 1) * 128)) + (db >> 1) * 256 : (off ^ (u * 64)) + db * 128;
            x.s[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(tile + at + (16 * t + 8 * u) * CH * 16));
        }
        return x.v;
    }
};

// The order of a tile's instructions: the compiler otherwise reads an operand from LDS right before the product that takes it, and one or two wavefronts a SIMD
// wait for most of these reads.
#define TENMO_READS(n) __builtin_amdgcn_sched_group_barrier(0x100, n, 0)
#define TENMO_PRODUCTS(n) __builtin_amdgcn_sched_group_barrier(0x008, n, 0)

// c += a b of 32 x 32 x 16 with both operands as halves
__device__ __forceinline__ void split_mfma(f32x16& c, f16x8 ah, f16x8 al, f16x8 bh, f16x8 bl) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, c, 0, 0, 0);
}
// two of them in turn: no product waits for the one before it
__device__ __forceinline__ void split_mfma2(f32x16& c, f16x8 ah, f16x8 al, f16x8 bh, f16x8 bl, f32x16& d, f16x8 eh, f16x8 el, f16x8 fh, f16x8 fl) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, c, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(el, fh, d, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, c, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(eh, fl, d, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, c, 0, 0, 0);
    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(eh, fh, d, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}
// registers 8 t .. 8 t + 7 of a product as an operand
__device__ __forceinline__ void halves(const f32x16& x, int t, float one, f16x8& h, f16x8& l) {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (_Float16)x[8 * t + e];
    // one h for both uses: left alone, the compiler may round a product that ends in x to fp16 by two ways that differ where x lies between two halves
    asm("" : "+v"(h));
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = (_Float16)__builtin_fmaf(x[8 * t + e], one, -(float)h[e]);
}
// row operand of the wavefront's own 32 rows, straight from memory
template <int DP>
__device__ __forceinline__ void own_rows(f16x8 (&h)[DP / 16], f16x8 (&l)[DP / 16], const float* rows, int lane) {
    const float* p = rows + (lane & 31) * DP + 8 * (lane >> 5);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        h[ks] = *(const f16x8*)(p + 16 * ks);
        l[ks] = *(const f16x8*)(p + 16 * ks + 4);
    }
}
// The same from the fp32 operand, a row a lane (and the other half of it 32 lanes further), each with a scale of its own, which is returned: a row of these is a column of the
// product, so none loses anything to another.  Rows that are not `in` are zeros.  *norm: the row's.
template <int DP>
__device__ __forceinline__ float own_split(f16x8 (&h)[DP / 16], f16x8 (&l)[DP / 16], const AttnOperand& o, int b, int i, int head, bool in, int D, float* norm) {
    constexpr int KD = DP / 16;
    const int half = (threadIdx.x & 63) >> 5;
    const float* p = o.p + b * o.b + (in ? i : 0) * o.s + head * o.h;
    f32x4 x[KD][2];
    float top = 0.f, sq = 0.f;
    attn_with_kind(attn_kind(o.d, D), [&](auto kind) {
#pragma unroll
        for (int ks = 0; ks < KD; ++ks)
#pragma unroll
            for (int u = 0; u < 2; ++u) x[ks][u] = attn_load4<kind.value>(p, o.d, 4 * ks + 2 * half + u, D);
    });
#pragma unroll
    for (int ks = 0; ks < KD; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[ks][u][e] = in ? x[ks][u][e] : 0.f; // whatever the row holds
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, __uint_as_float(finite_magnitude(x[ks][u][e])));
            sq += dot4(x[ks][u], x[ks][u]);
        }
    top = halves_max(top);
    sq = halves_sum(sq);
    *norm = sq < 1e37f && sq > 1e-30f ? sqrtf(sq) : fminf(top * sqrtf((float)D), 1e38f); // (a square out of range: the largest magnitude times sqrt(D) instead)
    const float scale = split_scale(__float_as_uint(top));
#pragma unroll
    for (int ks = 0; ks < KD; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 hi, lo;
            split_value(x[ks][e >> 2][e & 3] * scale, hi, lo);
            h[ks][e] = hi;
            l[ks][e] = lo;
        }
    return scale;
}
// register e of a product is row 8 (e / 4) + 4 (lane / 32) + e % 4
__device__ __forceinline__ int reg_row(int e) { return 8 * (e >> 2) + (e & 3); }

// A workgroup's head and block of rows.  Heads are dealt to the XCDs, so that one head's rows meet in one L2.  With a causal mask the blocks differ in length by the
// number of blocks: the longest of all heads come first ([8,1024,12,64]: CUs busy for 57 % of the launch when each head's blocks followed each other).
__device__ __forceinline__ void head_and_block(int id, int heads, int blocks, bool causal, bool last_is_longest, int* bh, int* block) {
    const bool deal = heads % 8 == 0;
    const int t = deal ? id / 8 : id, mine = deal ? heads / 8 : heads;
    const int h = causal ? t % mine : t / blocks, x = causal ? t / mine : t % blocks;
    *bh = __builtin_amdgcn_readfirstlane(deal ? id % 8 + 8 * h : h);
    *block = __builtin_amdgcn_readfirstlane(last_is_longest ? blocks - 1 - x : x);
}

// ---- forward -------------------------------------------------------------------------------------------------------------------------

template <int DP>
__global__ __launch_bounds__(256, 2) void attn_tile_forward_kernel(const TileArgs a) {
    using T = Tile<DP>;
    constexpr int STAGES = DP <= 64 ? 3 : 2, LOADS = 2 * T::BLOCKS / 4;
    __shared__ __align__(1024) float lds[STAGES * 2 * T::BYTES / 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, D = a.s.dim;
    const int pad_q = row_pad(a.s.queries), pad_k = row_pad(a.s.keys), q_blocks = pad_q / kRowPad;
    int bh, block;
    const int split = blockIdx.x % a.splits;
    head_and_block(blockIdx.x / a.splits, a.s.batch * a.s.heads, q_blocks, a.s.causal, true, &bh, &block);
    const int b = bh / a.s.heads, h = bh % a.s.heads, bk = b * a.s.kv_heads + h / a.s.group;
    const int length = __builtin_amdgcn_readfirstlane(attn_length(a.s, b)), start = __builtin_amdgcn_readfirstlane(attn_start(a.s, b));
    const int q0 = block * kRowPad + wave * 32, i = q0 + (lane & 31);
    const int limit = i < a.s.queries ? attn_limit(length, start, i) : 0;
    const int wave_last = q0 + 31 < a.s.queries ? q0 + 31 : a.s.queries - 1, block_last = (block + 1) * kRowPad < a.s.queries ? (block + 1) * kRowPad - 1 : a.s.queries - 1;
    const int wave_most = q0 < a.s.queries ? attn_limit(length, start, wave_last) : 0, wave_least = wave_last == q0 + 31 ? attn_limit(length, start, q0) : 0;
    const int tiles = (attn_limit(length, start, block_last) + 31) / 32, per = (tiles + a.splits - 1) / a.splits;
    const int t0 = split * per < tiles ? split * per : tiles, t1 = t0 + per < tiles ? t0 + per : tiles;

    if (__builtin_amdgcn_readfirstlane(keys_beyond(a, bk))) {
        constexpr int L = T::LANES;
        for (int r = q0; r < q0 + 32 && r < a.s.queries; ++r) {
            float m, l;
            const int most = attn_limit(length, start, r), hi = t1 * 32 < most ? t1 * 32 : most;
            const f32x4 o = slow_forward<L>(a, b, h, r, t0 * 32, hi, m, l);
            const int64_t row = (int64_t)bh * a.s.queries + r;
            if (lane >= L) continue;
            if (a.part) {
                float* to = a.part + ((int64_t)split * a.s.batch * a.s.heads * a.s.queries + row) * (D + 2);
                store_part(to, 4 * lane, D, o);
                if (lane == 0) to[D] = m, to[D + 1] = l;
            } else {
                store_part(a.to + (((int64_t)b * a.s.queries + r) * a.s.heads + h) * D, 4 * lane, D, l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o / l);
                if (lane == 0 && a.to_lse) a.to_lse[row] = l == 0.f ? kNone : m + logf(l);
            }
        }
        return;
    }
    f16x8 qh[T::KD], ql[T::KD];
    float norm_q;
    const float scale_q = own_split<DP>(qh, ql, a.src[kQ], b, i, h, limit > 0, D, &norm_q);
    const float c_all = fabsf(a.s.scale) * kLog2e / scale_q;
    const float *const scale_k = a.scale[kK] + (int64_t)bk * (pad_k / 64), *const scale_v = a.scale[kV] + (int64_t)bk * (pad_k / 64);
    int unit = 127 << 23; // the bits of the power of two that V is multiplied by in the sums
    float lane_k, lane_v; // of 64 blocks, one a lane
    auto load_scales = [&](int t) {
        const int i = (t >> 7) * 64 + lane < pad_k / 64 ? (t >> 7) * 64 + lane : 0;
        lane_k = scale_k[i];
        lane_v = scale_v[i];
        asm volatile("" : "+v"(lane_k), "+v"(lane_v)); // waited for here: a wait in every tile would be one for the tiles that are on their way
    };
    load_scales(t0);
    if (a.s.scale < 0.f) // the maximum is taken before the factor, which has to keep the order
#pragma unroll
        for (int ks = 0; ks < T::KD; ++ks) qh[ks] = -qh[ks], ql[ks] = -ql[ks];
    const float* const base[2] = {a.split[kK] + (int64_t)bk * pad_k * DP, a.split[kV] + (int64_t)bk * pad_k * DP};
    uint32_t off[LOADS];
    T::template offsets<2>(off, wave, lane);
    auto load = [&](int t, int stage) {
        const float* const src[2] = {base[0] + (int64_t)t * 32 * DP, base[1] + (int64_t)t * 32 * DP};
        T::template load<2>(lds, stage * 2 * T::BYTES, src, off, wave);
    };
    const uint32_t row_off[2] = {T::row_offset(lane, 0), T::row_offset(lane, 1)}, col_off[2] = {T::column_offset(lane, 0), T::column_offset(lane, 1)};

    const float one = variable_one();
    f32x16 o[T::ND];
#pragma unroll
    for (int d = 0; d < T::ND; ++d) o[d] = zero16();
    float m = kNone, l = 0.f;
    if (t0 < t1) load(t0, 0);
    if (STAGES == 3 && t0 + 1 < t1) load(t0 + 1, 1);
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
        if (STAGES == 3 && t + 1 < t1) stage_barrier<LOADS>();
        else stage_barrier<0>();
        if (t + STAGES - 1 < t1) load(t + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        const char* ks_tile = (const char*)lds + stage * 2 * T::BYTES;
        const char* vs_tile = ks_tile + T::BYTES;
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        if (t * 32 >= wave_most) continue; // nothing here for these 32 queries (every wavefront meets at the next barrier)
        if (t % 128 == 0) load_scales(t);
        // V of this block has a scale of its own: p makes up for it where that costs no more than 4 of its bits, else the sums do (by 2^16 at the most: keys_beyond())
        const float c = c_all * lane_value(lane_k, (t >> 1) & 63);
        const int own = __builtin_amdgcn_readlane(__float_as_int(lane_v), (t >> 1) & 63), scale = own ? own : unit, more = (scale - unit) >> 23;
        const bool other = more < 0 || more > 4;
        const float up = other ? __int_as_float((127 << 23) + scale - unit) : 1.f, less = kPBits - (other ? 0.f : (float)more), back = __int_as_float((127 + (other ? 0 : more)) << 23);
        unit = other ? scale : unit;
        f32x16 s = zero16();
#pragma unroll
        for (int ks = 0; ks < T::KD; ++ks) split_mfma(s, T::row_read(ks_tile, row_off[0], ks), T::row_read(ks_tile, row_off[1], ks), qh[ks], ql[ks]);
        TENMO_READS(4);
#pragma unroll
        for (int ks = 0; ks < T::KD - 2; ++ks) {
            TENMO_PRODUCTS(3);
            TENMO_READS(2);
        }
        TENMO_PRODUCTS(6);
        float by = c;
        if (t * 32 + 32 > wave_least) { // (the factor first: it may be 0, and -inf has to stay what it is)
            const int left = limit - t * 32 - 4 * half;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = reg_row(e) < left ? s[e] * c : kNone;
            by = 1.f;
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        top = halves_max(top) * by;
        if (__any(top > m + kRenew) || other) { // (an m of -inf is passed by any score)
            const float now = top > m + kRenew ? top : m, keep = m == kNone ? 0.f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= keep;
#pragma unroll
            for (int d = 0; d < T::ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= keep * up;
        }
        const float shift = less - (m == kNone ? 0.f : m);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(s[e] * by + shift);
            sum += s[e];
        }
        l += sum * back;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            f16x8 ph, pl;
            halves(s, t2, one, ph, pl);
#pragma unroll
            for (int d = 0; d < T::ND; ++d) split_mfma(o[d], T::column_read(vs_tile, col_off[0], t2, d), T::column_read(vs_tile, col_off[1], t2, d), ph, pl);
        }
        TENMO_READS(8);
#pragma unroll
        for (int x = 0; x < 2 * T::ND - 2; ++x) {
            TENMO_PRODUCTS(3);
            TENMO_READS(4);
        }
        TENMO_PRODUCTS(6);
    }
    l = halves_sum(l);
    if (i >= a.s.queries) return;
    const int64_t row = (int64_t)bh * a.s.queries + i;
    float* to;
    float factor;
    if (a.part) {
        to = a.part + ((int64_t)split * a.s.batch * a.s.heads * a.s.queries + row) * (D + 2);
        factor = 1.f / 128.f;
        if (half == 0) to[D] = m * kLn2, to[D + 1] = l * (1.f / 128.f);
    } else {
        to = a.to + (((int64_t)b * a.s.queries + i) * a.s.heads + h) * D;
        factor = l == 0.f ? 0.f : 1.f / l;
        // The 2^7 goes before the logarithm, which it would make larger and so coarser: an error here is one of all of the row's probabilities backward ([1,500..2000] 7e-7, so 3e-7)
        if (half == 0 && a.to_lse) a.to_lse[row] = l == 0.f ? kNone : fmaf(m, kLn2, logf(l * (1.f / 128.f)));
    }
    const float inv_v = power_inverse(__int_as_float(unit)); // (by itself: its product with the factor may be too small for a float)
#pragma unroll
    for (int d = 0; d < T::ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = 32 * d + 8 * q + 4 * half;
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[d][4 * q + e] * factor * inv_v;
            store_part(to, at, D, x);
        }
}

// ---- backward ------------------------------------------------------------------------------------------------------------------------

// The scale of what a lane's sums are made of: brings the largest so far into 2^10 .. 2^15
struct Unit {
    float scale = 0x1p126f, most = 0x1p-111f; // most: 2^15 / scale
    // for a larger one (of both halves of the wavefront); gives what the sums are to be multiplied by
    __device__ __forceinline__ float renew(float top) {
        const int e = (int)(__float_as_uint(top) >> 23) - 127; // of top: -111 .. 128 where it is too large
        const float now = top > most ? __uint_as_float((uint32_t)(10 - e + 127) << 23) : scale, by = now * power_inverse(scale);
        scale = now;
        most = 0x1p15f * power_inverse(now);
        return by;
    }
};

// Sums that lie in accumulation registers stay there: a plain product would have the compiler move them, or what it moves for them, in every tile (113 moves of 361 instructions at DP = 128).
// Before the first read: the wait states behind a matrix instruction that wrote them; behind the last write: those before one that reads them.
template <bool ACCUMULATION, int N>
__device__ __forceinline__ void scale_sums(f32x16 (&x)[N], float by) {
    if constexpr (ACCUMULATION) {
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float v = x[d][e], t;
                asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32_e32 %1, %2, %1\n\tv_accvgpr_write_b32 %0, %1" : "+a"(v), "=&v"(t) : "v"(by));
                x[d][e] = v;
            }
        asm volatile("s_nop 7" ::: "memory");
    } else {
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[d][e] *= by;
    }
}

__device__ __forceinline__ void store_gradient(const AttnOperand& g, int64_t at, int d, int D, f32x4 x, int accumulate) {
    float* to = g.p + at + d * g.d;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d + e < D) to[e * g.d] = accumulate ? to[e * g.d] + x[e] : x[e];
}

template <int DP>
struct Backward {
    static constexpr int STAGES = DP <= 64 ? 3 : 2, STAGE = 2 * Tile<DP>::BYTES + 1024; // two tiles, and what is known of the rows
};

template <int DP>
__device__ __forceinline__ void tile_dkv(const TileArgs& a, int id, float* lds) {
    using T = Tile<DP>;
    constexpr int STAGES = Backward<DP>::STAGES, STAGE = Backward<DP>::STAGE, LOADS = 2 * T::BLOCKS / 4 + 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, D = a.s.dim;
    const int pad_q = row_pad(a.s.queries), pad_k = row_pad(a.s.keys), k_blocks = pad_k / kRowPad;
    int bh, block;
    const int run = id % a.query_runs;
    head_and_block(id / a.query_runs, a.s.batch * a.s.heads, k_blocks, a.s.causal, false, &bh, &block);
    const int b = bh / a.s.heads, h = bh % a.s.heads, hk = h / a.s.group, bk = b * a.s.kv_heads + hk;
    const int length = __builtin_amdgcn_readfirstlane(attn_length(a.s, b)), start = __builtin_amdgcn_readfirstlane(attn_start(a.s, b)), keys = used_keys(a.s, length, start);
    const int j0 = block * kRowPad + wave * 32, j = j0 + (lane & 31);
    // query i sees key j when i >= j - start and j < length
    const int see = a.s.causal ? j - start : 0;
    const int block_first = a.s.causal && block * kRowPad - start > 0 ? block * kRowPad - start : 0;
    const int first = block_first / 32, end = block * kRowPad < keys ? (a.s.queries + 31) / 32 : 0, per = end > first ? (end - first + a.query_runs - 1) / a.query_runs : 0;
    const int t0 = first + run * per, t1 = t0 + per < end ? t0 + per : end;
    const int64_t run_at = (int64_t)run * a.s.batch * a.s.heads * a.s.keys * D;

    const f32x4 head_q = a.head[kQ][bh], head_k = a.head[kK][bk], head_v = a.head[kV][bk], head_g = a.head[kDO][bh];
    if (__builtin_amdgcn_readfirstlane(beyond(a, head_q, head_k, head_v) || head_g[2] > 0.f)) {
        constexpr int L = T::LANES;
        for (int r = lane / L; r < 32 && __any(j0 + r < a.s.keys); r += 64 / L) {
            f32x4 x, y;
            const int key = j0 + r, d = 4 * (lane % L);
            slow_dkv<L>(a, b, h, key, length, start, t0 * 32, t1 * 32 < a.s.queries ? t1 * 32 : a.s.queries, x, y);
            if (key >= a.s.keys) continue;
            x *= a.s.scale;
            if (a.part_k) {
                store_part(a.part_k + run_at + ((int64_t)bh * a.s.keys + key) * D, d, D, x);
                store_part(a.part_v + run_at + ((int64_t)bh * a.s.keys + key) * D, d, D, y);
                continue;
            }
            if (a.grad_k.p) store_gradient(a.grad_k, b * a.grad_k.b + hk * a.grad_k.h + key * a.grad_k.s, d, D, x, a.accumulate);
            if (a.grad_v.p) store_gradient(a.grad_v, b * a.grad_v.b + hk * a.grad_v.h + key * a.grad_v.s, d, D, y, a.accumulate);
        }
        return;
    }
    f16x8 kh[T::KD], kl[T::KD], vh[T::KD], vl[T::KD];
    own_rows<DP>(kh, kl, a.split[kK] + ((int64_t)bk * pad_k + j0) * DP, lane);
    own_rows<DP>(vh, vl, a.split[kV] + ((int64_t)bk * pad_k + j0) * DP, lane);
    const float scale_q = head_q[0], scale_g = head_g[0];
    const float c = a.s.scale * kLog2e / scale_q / head_k[0], inv_dp = 1.f / scale_g / head_v[0];
    const float* const base[2] = {a.split[kQ] + (int64_t)bh * pad_q * DP, a.split[kDO] + (int64_t)bh * pad_q * DP};
    const float* const stats = a.stats + (int64_t)bh * pad_q * kStats;
    uint32_t off[LOADS - 1];
    T::template offsets<2>(off, wave, lane);
    auto load = [&](int t, int stage) {
        const float* const src[2] = {base[0] + (int64_t)t * 32 * DP, base[1] + (int64_t)t * 32 * DP};
        T::template load<2>(lds, stage * STAGE, src, off, wave);
        // the tile's 32 rows, and the 32 behind them, which are not used: every wavefront brings the same
        direct_load_16B(lds, stage * STAGE + 2 * T::BYTES, lane * 16, stats + (int64_t)t * (32 * kStats));
    };
    const uint32_t row_off[2] = {T::row_offset(lane, 0), T::row_offset(lane, 1)}, col_off[2] = {T::column_offset(lane, 0), T::column_offset(lane, 1)};

    const float one = variable_one();
    f32x16 dk[T::ND], dv[T::ND];
#pragma unroll
    for (int d = 0; d < T::ND; ++d) dk[d] = dv[d] = zero16();
    Unit unit_p, unit_s;
    if (t0 < t1) load(t0, 0);
    if (STAGES == 3 && t0 + 1 < t1) load(t0 + 1, 1);
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
        if (STAGES == 3 && t + 1 < t1) stage_barrier<LOADS>();
        else stage_barrier<0>();
        if (t + STAGES - 1 < t1) load(t + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        const char* q_tile = (const char*)lds + stage * STAGE;
        const char* g_tile = q_tile + T::BYTES;
        const f32x4* st = (const f32x4*)(g_tile + T::BYTES) + half; // four rows each
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        const int i0 = t * 32;

        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int ks = 0; ks < T::KD; ++ks) {
            split_mfma2(s, T::row_read(q_tile, row_off[0], ks), T::row_read(q_tile, row_off[1], ks), kh[ks], kl[ks],
                        dp, T::row_read(g_tile, row_off[0], ks), T::row_read(g_tile, row_off[1], ks), vh[ks], vl[ks]);
        }
        f32x4 lse[4], delta[4]; // of the rows 8 q + 4 half + 0..3
#pragma unroll
        for (int q = 0; q < 4; ++q) lse[q] = st[8 * kLseUp + 2 * q], delta[q] = st[8 * kDeltaUp + 2 * q];
        TENMO_READS(8);
#pragma unroll
        for (int ks = 0; ks < T::KD - 2; ++ks) {
            TENMO_PRODUCTS(6);
            TENMO_READS(4);
        }
        TENMO_PRODUCTS(6);
        TENMO_READS(8);
        TENMO_PRODUCTS(6);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = s[e] * c - lse[e >> 2][e & 3];
            dp[e] = dp[e] * inv_dp - delta[e >> 2][e & 3];
        }
        if (i0 < j0 + 31 - start || j0 + 32 > length) { // some pairs are not allowed: their p is 0, whatever the rest
            const int from = j < length ? see - i0 - 4 * half : 32;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool ok = reg_row(e) >= from;
                s[e] = ok ? s[e] : kNone;
                dp[e] = ok ? dp[e] : 0.f;
            }
        }
        float top_p = 0.f, top_s = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(s[e]);
            dp[e] *= s[e];
            top_p = fmaxf(top_p, s[e]);
            top_s = fmaxf(top_s, fabsf(dp[e]));
        }
        top_p = halves_max(top_p);
        top_s = halves_max(top_s);
        if (__any(top_p > unit_p.most || top_s > unit_s.most)) {
            if (__any(top_p > unit_p.most)) scale_sums<(DP > 64)>(dv, unit_p.renew(top_p));
            if (__any(top_s > unit_s.most)) scale_sums<(DP > 64)>(dk, unit_s.renew(top_s));
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= unit_p.scale, dp[e] *= unit_s.scale;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            f16x8 ph, pl, sh, sl;
            halves(s, t2, one, ph, pl);
            halves(dp, t2, one, sh, sl);
#pragma unroll
            for (int d = 0; d < T::ND; ++d) {
                split_mfma2(dv[d], T::column_read(g_tile, col_off[0], t2, d), T::column_read(g_tile, col_off[1], t2, d), ph, pl,
                            dk[d], T::column_read(q_tile, col_off[0], t2, d), T::column_read(q_tile, col_off[1], t2, d), sh, sl);
            }
        }
        TENMO_READS(16);
#pragma unroll
        for (int x = 0; x < 2 * T::ND - 2; ++x) {
            TENMO_PRODUCTS(6);
            TENMO_READS(8);
        }
        TENMO_PRODUCTS(12);
    }
    if (j >= a.s.keys) return;
    const float inv_ds = power_inverse(unit_s.scale), inv_q = 1.f / scale_q, inv_p = power_inverse(unit_p.scale), inv_g = 1.f / scale_g; // (one after the other: their product may be too small for a float)
    const int64_t at_k = b * a.grad_k.b + hk * a.grad_k.h + j * a.grad_k.s, at_v = b * a.grad_v.b + hk * a.grad_v.h + j * a.grad_v.s;
    const int64_t at_part = run_at + ((int64_t)bh * a.s.keys + j) * D;
#pragma unroll
    for (int d = 0; d < T::ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = 32 * d + 8 * q + 4 * half;
            f32x4 x, y;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = dk[d][4 * q + e] * a.s.scale * inv_q * inv_ds, y[e] = dv[d][4 * q + e] * inv_p * inv_g;
            if (a.part_k) {
                store_part(a.part_k + at_part, at, D, x);
                store_part(a.part_v + at_part, at, D, y);
                continue;
            }
            if (a.grad_k.p) store_gradient(a.grad_k, at_k, at, D, x, a.accumulate);
            if (a.grad_v.p) store_gradient(a.grad_v, at_v, at, D, y, a.accumulate);
        }
}

template <int DP>
__device__ __forceinline__ void tile_dq(const TileArgs& a, int id, float* lds) {
    using T = Tile<DP>;
    constexpr int STAGES = Backward<DP>::STAGES, LOADS = 2 * T::BLOCKS / 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, D = a.s.dim;
    const int pad_q = row_pad(a.s.queries), pad_k = row_pad(a.s.keys), q_blocks = pad_q / kRowPad;
    int bh, block;
    const int run = id % a.key_runs;
    head_and_block(id / a.key_runs, a.s.batch * a.s.heads, q_blocks, a.s.causal, true, &bh, &block);
    const int b = bh / a.s.heads, h = bh % a.s.heads, bk = b * a.s.kv_heads + h / a.s.group;
    const int length = __builtin_amdgcn_readfirstlane(attn_length(a.s, b)), start = __builtin_amdgcn_readfirstlane(attn_start(a.s, b));
    const int q0 = block * kRowPad + wave * 32, i = q0 + (lane & 31);
    const int limit = i < a.s.queries ? attn_limit(length, start, i) : 0;
    const int wave_last = q0 + 31 < a.s.queries ? q0 + 31 : a.s.queries - 1, block_last = (block + 1) * kRowPad < a.s.queries ? (block + 1) * kRowPad - 1 : a.s.queries - 1;
    const int wave_least = wave_last == q0 + 31 ? attn_limit(length, start, q0) : 0;
    const int tiles = (attn_limit(length, start, block_last) + 31) / 32, per = (tiles + a.key_runs - 1) / a.key_runs;
    const int t0 = run * per < tiles ? run * per : tiles, t1 = t0 + per < tiles ? t0 + per : tiles;
    float* const part = a.part_q ? a.part_q + ((int64_t)run * a.s.batch * a.s.heads + bh) * a.s.queries * D : nullptr;

    const f32x4 head_q = a.head[kQ][bh], head_k = a.head[kK][bk], head_v = a.head[kV][bk], head_g = a.head[kDO][bh];
    if (__builtin_amdgcn_readfirstlane(beyond(a, head_q, head_k, head_v) || head_g[2] > 0.f)) {
        constexpr int L = T::LANES;
        for (int r = q0; r < q0 + 32 && r < a.s.queries; ++r) {
            const int most = attn_limit(length, start, r), hi = t1 * 32 < most ? t1 * 32 : most;
            const f32x4 x = slow_dq<L>(a, b, h, r, t0 * 32, hi, a.lse[(int64_t)bh * a.s.queries + r], a.stats[stat_at((int64_t)bh * pad_q + r, kDelta)]);
            if (part && lane < L) store_part(part + (int64_t)r * D, 4 * lane, D, x * a.s.scale);
            else if (lane < L) store_gradient(a.grad_q, b * a.grad_q.b + h * a.grad_q.h + r * a.grad_q.s, 4 * lane, D, x * a.s.scale, a.accumulate);
        }
        return;
    }
    f16x8 qh[T::KD], ql[T::KD], gh[T::KD], gl[T::KD];
    own_rows<DP>(qh, ql, a.split[kQ] + ((int64_t)bh * pad_q + q0) * DP, lane);
    own_rows<DP>(gh, gl, a.split[kDO] + ((int64_t)bh * pad_q + q0) * DP, lane);
    const float scale_k = head_k[0];
    const float lse2 = limit > 0 ? a.lse[(int64_t)bh * a.s.queries + i] * kLog2e : __builtin_inff(), delta = a.stats[stat_at((int64_t)bh * pad_q + i, kDelta)];
    const float c = a.s.scale * kLog2e / head_q[0] / scale_k, inv_dp = 1.f / head_g[0] / head_v[0] * a.stats[stat_at((int64_t)bh * pad_q + i, kDown)];
    const float* const base[2] = {a.split[kK] + (int64_t)bk * pad_k * DP, a.split[kV] + (int64_t)bk * pad_k * DP};
    uint32_t off[LOADS];
    T::template offsets<2>(off, wave, lane);
    auto load = [&](int t, int stage) {
        const float* const src[2] = {base[0] + (int64_t)t * 32 * DP, base[1] + (int64_t)t * 32 * DP};
        T::template load<2>(lds, stage * 2 * T::BYTES, src, off, wave);
    };
    const uint32_t row_off[2] = {T::row_offset(lane, 0), T::row_offset(lane, 1)}, col_off[2] = {T::column_offset(lane, 0), T::column_offset(lane, 1)};

    const float one = variable_one();
    f32x16 dq[T::ND];
#pragma unroll
    for (int d = 0; d < T::ND; ++d) dq[d] = zero16();
    Unit unit;
    if (t0 < t1) load(t0, 0);
    if (STAGES == 3 && t0 + 1 < t1) load(t0 + 1, 1);
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
        if (STAGES == 3 && t + 1 < t1) stage_barrier<LOADS>();
        else stage_barrier<0>();
        if (t + STAGES - 1 < t1) load(t + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        const char* k_tile = (const char*)lds + stage * 2 * T::BYTES;
        const char* v_tile = k_tile + T::BYTES;
        stage = stage == STAGES - 1 ? 0 : stage + 1;

        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int ks = 0; ks < T::KD; ++ks) {
            split_mfma2(s, T::row_read(k_tile, row_off[0], ks), T::row_read(k_tile, row_off[1], ks), qh[ks], ql[ks],
                        dp, T::row_read(v_tile, row_off[0], ks), T::row_read(v_tile, row_off[1], ks), gh[ks], gl[ks]);
        }
        TENMO_READS(8);
#pragma unroll
        for (int ks = 0; ks < T::KD - 2; ++ks) {
            TENMO_PRODUCTS(6);
            TENMO_READS(4);
        }
        TENMO_PRODUCTS(12);
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = __builtin_amdgcn_exp2f(s[e] * c - lse2) * (dp[e] * inv_dp - delta);
        if (t * 32 + 32 > wave_least) {
            const int left = limit - t * 32 - 4 * half;
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = reg_row(e) < left ? dp[e] : 0.f;
        }
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(dp[e]));
        top = halves_max(top);
        if (__any(top > unit.most)) {
            scale_sums<(DP > 64)>(dq, unit.renew(top));
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] *= unit.scale;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            f16x8 sh, sl;
            halves(dp, t2, one, sh, sl);
#pragma unroll
            for (int d = 0; d < T::ND; ++d) split_mfma(dq[d], T::column_read(k_tile, col_off[0], t2, d), T::column_read(k_tile, col_off[1], t2, d), sh, sl);
        }
        TENMO_READS(8);
#pragma unroll
        for (int x = 0; x < 2 * T::ND - 2; ++x) {
            TENMO_PRODUCTS(3);
            TENMO_READS(4);
        }
        TENMO_PRODUCTS(6);
    }
    if (i >= a.s.queries) return;
    const float inv_ds = power_inverse(unit.scale), inv_k = 1.f / scale_k;
    const int64_t at_q = b * a.grad_q.b + h * a.grad_q.h + i * a.grad_q.s;
#pragma unroll
    for (int d = 0; d < T::ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = dq[d][4 * q + e] * a.s.scale * inv_k * inv_ds;
            if (part) store_part(part + (int64_t)i * D, 32 * d + 8 * q + 4 * half, D, x);
            else store_gradient(a.grad_q, at_q, 32 * d + 8 * q + 4 * half, D, x, a.accumulate);
        }
}

// Both in one launch, the blocks of keys (four products a tile) before the blocks of queries (three): neither needs the other, and the ends of the first, when the chip empties, are filled by the second.
template <int DP>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void attn_tile_backward_kernel(const TileArgs a, int key_blocks) {
    __shared__ __align__(1024) float lds[Backward<DP>::STAGES * Backward<DP>::STAGE / 4];
    if ((int)blockIdx.x < key_blocks) tile_dkv<DP>(a, blockIdx.x, lds);
    else tile_dq<DP>(a, blockIdx.x - key_blocks, lds);
}

// The parts of dK, dV (of the query heads that share a key head) and dQ, in order: blockIdx.y.  [1,8192,16/4,128], two runs of each: 107 us for 540 MB.
__global__ __launch_bounds__(256) void attn_parts_kernel(const TileArgs a) {
    const int D = a.s.dim, quads = (D + 3) / 4, which = blockIdx.y;
    const bool keys = which < 2;
    const float* __restrict part = which == 0 ? a.part_k : which == 1 ? a.part_v : a.part_q;
    const AttnOperand g{which == 0 ? a.grad_k.p : which == 1 ? a.grad_v.p : a.grad_q.p, which == 0 ? a.grad_k.b : which == 1 ? a.grad_v.b : a.grad_q.b,
                        which == 0 ? a.grad_k.s : which == 1 ? a.grad_v.s : a.grad_q.s, which == 0 ? a.grad_k.h : which == 1 ? a.grad_v.h : a.grad_q.h,
                        which == 0 ? a.grad_k.d : which == 1 ? a.grad_v.d : a.grad_q.d};
    if (!g.p || !part) return;
    const int heads = keys ? a.s.kv_heads : a.s.heads, rows = keys ? a.s.keys : a.s.queries, group = keys ? a.s.group : 1, runs = keys ? a.query_runs : a.key_runs;
    const int64_t all = (int64_t)a.s.batch * heads * rows * quads, run_at = (int64_t)a.s.batch * a.s.heads * rows * D;
    attn_with_kind(attn_kind(1, D), [&](auto kind) {
        for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < all; x += (int64_t)gridDim.x * 256) {
            const int d = (int)(x % quads) * 4;
            const int64_t row = x / quads, bh = row / rows, j = row - bh * rows, b = bh / heads, hk = bh - b * heads;
            const float* p = part + ((b * a.s.heads + hk * group) * rows + j) * D;
            f32x4 sum{0.f, 0.f, 0.f, 0.f};
            for (int run = 0; run < runs; ++run) {
#pragma unroll 4
                for (int i = 0; i < group; ++i) sum += attn_load4<decltype(kind)::value>(p + run * run_at + (int64_t)i * rows * D, 1, d / 4, D);
            }
            store_gradient(g, b * g.b + hk * g.h + j * g.s, d, D, sum, a.accumulate);
        }
    });
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------

int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128; }

void plan_keys(TileArgs& a, Workspace& ws) {
    const AttnShape& s = a.s;
    const int64_t heads = (int64_t)s.batch * s.kv_heads, blocks = row_pad(s.keys) / 64;
    for (int j = 0; j < 2; ++j) {
        a.split[j] = ws.take<float>(heads * row_pad(s.keys) * padded_dim(s.dim));
        a.seen[j] = ws.take<f32x4>(heads * blocks);
        a.scale[j] = ws.take<float>(heads * blocks);
    }
}

int all_heads(const AttnShape& s) { return 2 * s.batch * (s.heads + s.kv_heads); }

void plan_operands(TileArgs& a, Workspace& ws) {
    const AttnShape& s = a.s;
    // Runs of 128 rows, or, where that is fewer than four workgroups a CU, of the rows that one has in flight at once ([8,1024,12,64]: 259 us, 256 with 128 rows); no more than a launch holds.
    const int longest = std::max(s.queries, s.keys), once = 1024 / (s.dim <= 32 ? 8 : s.dim <= 64 ? 16 : 32);
    const int run = (int64_t)all_heads(s) * ((longest + 127) / 128) < 1024 ? once : 128;
    a.parts = std::max(1, std::min(std::min(kHeadParts, (1 << 23) / all_heads(s)), (longest + run - 1) / run));
    for (int j = 0; j < 4; ++j) {
        const bool key = j == kK || j == kV;
        const int64_t heads = (int64_t)s.batch * (key ? s.kv_heads : s.heads);
        a.split[j] = ws.take<float>(heads * row_pad(key ? s.keys : s.queries) * padded_dim(s.dim));
        a.seen[j] = ws.take<f32x4>(heads * a.parts);
        a.head[j] = ws.take<f32x4>(heads);
    }
}

template <int DP, int L>
void launch_forward(const TileArgs& a, hipStream_t stream) {
    const AttnShape& s = a.s;
    hipLaunchKernelGGL((attn_prepare_kernel<DP, L>), dim3((unsigned)(2 * s.batch * s.kv_heads * (row_pad(s.keys) / 64))), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(attn_tile_forward_kernel<DP>, dim3((unsigned)(s.batch * s.heads * (row_pad(s.queries) / kRowPad) * a.splits)), dim3(256), 0, stream, a);
}

template <int DP, int L>
void launch_backward(const TileArgs& a, hipStream_t stream) {
    const AttnShape& s = a.s;
    const int64_t rows = 2LL * s.batch * ((int64_t)s.heads * row_pad(s.queries) + (int64_t)s.kv_heads * row_pad(s.keys));
    hipLaunchKernelGGL(attn_amax_kernel<L>, dim3((unsigned)(all_heads(s) * a.parts)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(attn_split_kernel<DP>, dim3((unsigned)(rows / 64)), dim3(256), 0, stream, a);
    const int blocks_of_keys = a.grad_k.p || a.grad_v.p ? s.batch * s.heads * (row_pad(s.keys) / kRowPad) * a.query_runs : 0;
    const int blocks_of_queries = a.grad_q.p ? s.batch * s.heads * (row_pad(s.queries) / kRowPad) * a.key_runs : 0;
    hipLaunchKernelGGL(attn_tile_backward_kernel<DP>, dim3((unsigned)(blocks_of_keys + blocks_of_queries)), dim3(256), 0, stream, a, blocks_of_keys);
    const bool keys = a.part_k && blocks_of_keys, queries = a.part_q && blocks_of_queries;
    if (keys || queries) {
        const int64_t quads = (int64_t)s.batch * ((s.dim + 3) / 4) * std::max(keys ? (int64_t)s.kv_heads * s.keys : 0, queries ? (int64_t)s.heads * s.queries : 0);
        hipLaunchKernelGGL(attn_parts_kernel, dim3((unsigned)std::min<int64_t>((quads + 255) / 256, 4096), queries ? 3 : 2), dim3(256), 0, stream, a);
    }
}

} // namespace

void attn_tiles_forward(const AttnShape& s, const AttnOperand& q, const AttnOperand& k, const AttnOperand& v, float* out, float* lse,
                        Workspace& ws, int cus, hipStream_t stream, bool launch) {
    TileArgs a{};
    a.s = s;
    a.src[kQ] = q; a.src[kK] = k; a.src[kV] = v;
    a.to = out; a.to_lse = lse;
    plan_keys(a, ws);
    // two workgroups a CU fill it; a run of fewer than 256 keys is not worth its part of the join
    const int64_t groups = (int64_t)s.batch * s.heads * (row_pad(s.queries) / kRowPad);
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>(2LL * cus / groups, std::min(s.keys / 256, kMostRuns)));
    if (a.splits > 1) a.part = ws.take<float>((int64_t)a.splits * s.batch * s.heads * s.queries * (s.dim + 2));
    if (!launch) return;
    switch (padded_dim(s.dim)) {
        case 32: launch_forward<32, 8>(a, stream); break;
        case 64: launch_forward<64, 16>(a, stream); break;
        case 96: launch_forward<96, 32>(a, stream); break;
        default: launch_forward<128, 32>(a, stream);
    }
    if (a.splits > 1) attn_join(s, a.part, a.splits, out, lse, stream);
}

void attn_tiles_backward(const AttnBackward& b, Workspace& ws, int cus, hipStream_t stream, bool launch) {
    TileArgs a{};
    a.s = b.s;
    a.src[kQ] = b.q; a.src[kK] = b.k; a.src[kV] = b.v;
    a.src[kDO] = AttnOperand{const_cast<float*>(b.dout), (int64_t)b.s.queries * b.s.heads * b.s.dim, (int64_t)b.s.heads * b.s.dim, b.s.dim, 1};
    a.out = b.out; a.lse = b.lse;
    a.grad_q = b.grad_q; a.grad_k = b.grad_k; a.grad_v = b.grad_v; a.accumulate = b.accumulate;
    plan_operands(a, ws);
    a.stats = ws.take<float>(kStats * ((int64_t)b.s.batch * b.s.heads * row_pad(b.s.queries) + kRowPad));
    // A sum over many tiles is cut into runs, whose parts are added afterwards in order, for two reasons.  Few heads with few blocks leave CUs without a workgroup: runs are no longer than what three
    // workgroups a CU would do if all tiles were dealt evenly (a tile of queries for a block of keys is four products, one of keys for a block of queries three), and 8 tiles at least, or the parts
    // cost more.  Whole sums: [1,8192,8,64] for 500 keys 427 us, [1,2048,4,64] causal 121 us, [1,3000,6/2,128] 420 us; in runs 147, 66 and 386; with two workgroups a CU 141, 72 and 420, with four
    // 149, 68 and 375.  And the accumulators round at each product, three for 16 rows: dK of 8192 queries has an error of 1.2e-6 of itself (2-norm) in one sum, and 0.9e-6 in runs of 128 tiles at the
    // most; those cost 4 to 6 % ([1,8192,16/4,128] causal 2750 -> 2890 us).  No more than four of them for this, since their parts take memory.
    const double heads = (double)b.s.batch * b.s.heads, query_tiles = (b.s.queries + 31) / 32, key_tiles = (b.s.keys + 31) / 32;
    const double even = std::max(8.0, heads * (row_pad(b.s.keys) / kRowPad * query_tiles * 4.0 / 3.0 + row_pad(b.s.queries) / kRowPad * key_tiles) / (3.0 * cus));
    auto runs = [&](double tiles) { return (int)std::max({1.0, tiles / even, std::min(4.0, std::ceil(tiles / 128))}); };
    a.query_runs = runs(query_tiles);
    a.key_runs = runs(key_tiles);
    if (b.s.group > 1 || a.query_runs > 1) {
        a.part_k = ws.take<float>(a.query_runs * (int64_t)b.s.batch * b.s.heads * b.s.keys * b.s.dim);
        a.part_v = ws.take<float>(a.query_runs * (int64_t)b.s.batch * b.s.heads * b.s.keys * b.s.dim);
    }
    if (a.key_runs > 1) a.part_q = ws.take<float>(a.key_runs * (int64_t)b.s.batch * b.s.heads * b.s.queries * b.s.dim);
    if (!launch) return;
    switch (padded_dim(b.s.dim)) {
        case 32: launch_backward<32, 8>(a, stream); break;
        case 64: launch_backward<64, 16>(a, stream); break;
        case 96: launch_backward<96, 32>(a, stream); break;
        default: launch_backward<128, 32>(a, stream);
    }
}

} // namespace tenmo
