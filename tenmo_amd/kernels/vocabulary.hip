// Cross-entropy of the logits x = H W + bias over a vocabulary, from the hidden states (include/tenmo_hip_transformer.h).
//
//   lse = log sum_v exp(x_v),  loss = (1 - ls) (lse - x_t) + ls (lse - mean_v x_v)
//   G = (exp(x - lse) - (1 - ls) [v = t] - ls / V) [t valid],  scale_m = the upstream gradient of row m
//   dH = scale (G W^T),  dW = (scale H)^T G,  db = sum_m scale_m G
//
// Bound: the matrix units, 2 M V D flop forward, 6 M V D backward (the logits again, dH, dW).  All three products run as split fp16 products
// (split_gemm.hpp).
//   * forward: tiles of 256 words x 128 tokens; the words of a token lie in the registers of two lanes, so that a tile's maximum and sum of a token take
//     one exchange, and 8 bytes a token and tile leave the chip instead of 1 KiB of logits.  A second launch joins the tiles of a token in a fixed order.
//   * backward: a piece of the vocabulary at a time; the tiles of the first launch end as G in split form (|G| <= 1, so its scale is known beforehand: 2^14),
//     which the second launch multiplies with W and with H.  The piece is as large as 512 MiB of G allow.
#include "split_gemm.hpp"

#include <algorithm>

namespace tenmo {
namespace {

constexpr float kGScale = 16384.f;
constexpr int64_t kPieceValues = 128 << 20; // of G, 4 bytes each

struct Source { // an operand in the order in which it is split: rows x cols
    const float* p;
    int64_t rows, cols, rs, cs;
    const float* row_scale; // NULL: 1
};

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

// ---- amax and split -------------------------------------------------------------------------------------------------------------

struct SplitJobs {
    Source src[2];
    uint32_t* amax[2]; // kAmaxParts partial maxima
    SplitMatrix dst[2];
};

__global__ __launch_bounds__(256) void vocab_amax_kernel(const SplitJobs j) {
    __shared__ uint32_t slots[4];
    const Source& s = j.src[blockIdx.y];
    uint32_t top = 0;
    for (int64_t r = blockIdx.x; r < s.rows; r += kAmaxParts) {
        const float scale = s.row_scale ? s.row_scale[r] : 1.f;
        const float* p = s.p + r * s.rs;
        int64_t c = threadIdx.x * 4;
        if (s.cs == 1)
            for (; c + 3 < s.cols; c += 1024) {
                const f32x4 x = *(const f32x4_u*)(p + c) * scale;
                for (int e = 0; e < 4; ++e) top = max(top, finite_magnitude(x[e]));
            }
        for (; c < s.cols; c += 1024)
            for (int e = 0; e < 4 && c + e < s.cols; ++e) top = max(top, finite_magnitude(p[(c + e) * s.cs] * scale));
    }
    top = wave_max_bits(top);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) j.amax[blockIdx.y][blockIdx.x] = max(max(slots[0], slots[1]), max(slots[2], slots[3]));
}

// the scale of a matrix, from its partial maxima, in every thread of a workgroup of 256
__device__ __forceinline__ float scale_from(const uint32_t* __restrict amax, uint32_t* slots) {
    uint32_t top = 0;
    for (int i = threadIdx.x; i < kAmaxParts; i += 256) top = max(top, amax[i]);
    top = wave_max_bits(top);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = top;
    __syncthreads();
    return split_scale(max(max(slots[0], slots[1]), max(slots[2], slots[3])));
}

__global__ __launch_bounds__(256) void vocab_split_kernel(const SplitJobs j) {
    __shared__ uint32_t slots[4];
    const Source& s = j.src[blockIdx.y];
    const SplitMatrix& d = j.dst[blockIdx.y];
    const float scale = scale_from(j.amax[blockIdx.y], slots);
    const int64_t groups = d.pitch / 8, all = split_pad(s.rows) * groups;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / groups, c = (i - r * groups) * 8;
        f16x8 h, l;
        float x[8];
        if (r < s.rows && s.cs == 1 && c + 7 < s.cols) {
            const f32x4 a = *(const f32x4_u*)(s.p + r * s.rs + c), b = *(const f32x4_u*)(s.p + r * s.rs + c + 4);
            for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
        } else {
            for (int e = 0; e < 8; ++e) x[e] = r < s.rows && c + e < s.cols ? s.p[r * s.rs + (c + e) * s.cs] : 0.f;
        }
        const float rscale = r < s.rows && s.row_scale ? s.row_scale[r] : 1.f;
        for (int e = 0; e < 8; ++e) {
            _Float16 hi, lo;
            split_value(x[e] * rscale * scale, hi, lo);
            h[e] = hi;
            l[e] = lo;
        }
        float* to = d.p + r * d.pitch + c;
        *(f16x8*)to = h;
        *(f16x8*)(to + 4) = l;
    }
}

// ---- the products --------------------------------------------------------------------------------------------------------------------

struct ProductArgs {
    SplitMatrix a, b;
    const uint32_t *amax_a, *amax_b; // NULL: G, whose scale is kGScale
    int64_t M, N, k_steps;
    int64_t tiles_m, tiles_n;
};

struct LogitArgs {
    VocabArgs v;
    int64_t first; // word of the piece's first row
    int64_t words; // of the piece
    // forward
    float2* part;      // [tile][token]: maximum and sum
    float* part_x;     // [tile][token]: sum of the logits, with label smoothing
    float* target_logit; // [token]
    // backward
    const float* lse;
    const float* row_scale;
    SplitMatrix g;
    float* part_db; // [2 * token tiles][V], with a wanted bias gradient
};

template <bool A_KMAJOR, bool GRAD>
__global__ __launch_bounds__(256, 2) void vocab_logits_kernel(const ProductArgs p, const LogitArgs a) {
    __shared__ __align__(1024) float lds[kStages * kStageBytes / 4];
    __shared__ uint32_t slots[2][4];
    int64_t tm, tn;
    tile_of(blockIdx.x, (uint32_t)p.tiles_m, (uint32_t)p.tiles_n, &tm, &tn);
    const int64_t m0 = tm * kTileM, n0 = tn * kTileN;
    f32x16 acc[4][2];
    split_tile<A_KMAJOR, true>(acc, lds, p.a, m0, p.M, p.b, n0, p.N, p.k_steps);
    const float inv = 1.f / scale_from(p.amax_a, slots[0]) / scale_from(p.amax_b, slots[1]);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int64_t v0 = m0 + (wave & 1) * 128 + 4 * half; // of the piece; register e of block i is v0 + 32 i + 8 (e / 4) + e % 4
    // logits in place
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4 bias{0.f, 0.f, 0.f, 0.f};
            if (a.v.bias)
                for (int e = 0; e < 4; ++e) {
                    const int64_t v = v0 + 32 * i + 8 * q + e;
                    bias[e] = v < a.words ? a.v.bias[a.first + v] : 0.f;
                }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j][4 * q + e] = acc[i][j][4 * q + e] * inv + bias[e];
        }
    const bool edge = m0 + kTileM > a.words;
    if (!GRAD) {
        __shared__ float join[2][kTileN][3];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = (wave >> 1) * 64 + 32 * j + (lane & 31);
            const int64_t token = n0 + col;
            float top = -__builtin_inff(), sum = 0.f, sx = 0.f;
            if (edge) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const bool in = v0 + 32 * i + 8 * (e >> 2) + (e & 3) < a.words;
                        sx += in ? acc[i][j][e] : 0.f;
                        acc[i][j][e] = in ? acc[i][j][e] : -__builtin_inff();
                    }
            } else if (a.part_x) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sx += acc[i][j][e];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) sum += __expf(acc[i][j][e] - base);
            sum += __shfl_xor(sum, 32, 64);
            sx += __shfl_xor(sx, 32, 64);
            if (token < a.v.M) {
                const int64_t at = target_of(a.v, token) - a.first - v0; // target's place in this lane's words
                if (at >= 0 && at < 128) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (at == 32 * i + 8 * (e >> 2) + (e & 3)) a.target_logit[token] = acc[i][j][e];
                }
            }
            if ((wave & 1) && half == 0) join[0][col][0] = top, join[0][col][1] = sum, join[0][col][2] = sx;
            if (!(wave & 1) && half == 0) join[1][col][0] = top, join[1][col][1] = sum, join[1][col][2] = sx;
        }
        __syncthreads();
        if (threadIdx.x < kTileN && n0 + threadIdx.x < a.v.M) {
            const float *x = join[1][threadIdx.x], *y = join[0][threadIdx.x];
            const float top = fmaxf(x[0], y[0]), base = top == -__builtin_inff() ? 0.f : top;
            a.part[tm * a.v.M + n0 + threadIdx.x] = make_float2(top, x[1] * __expf(x[0] - base) + y[1] * __expf(y[0] - base));
            if (a.part_x) a.part_x[tm * a.v.M + n0 + threadIdx.x] = x[2] + y[2];
        }
    } else {
        const float smooth = a.v.ls / (float)a.v.V;
        float db[64];
        if (a.part_db)
#pragma unroll
            for (int x = 0; x < 64; ++x) db[x] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t token = n0 + (wave >> 1) * 64 + 32 * j + (lane & 31);
            const int64_t t = token < a.v.M ? target_of(a.v, token) : a.v.ignore;
            const bool valid = token < a.v.M && t != a.v.ignore;
            const float lse = valid ? a.lse[token] : 0.f, row_scale = valid ? a.row_scale[token] : 0.f;
            const int64_t at = t - a.first - v0;
            const bool store = token < split_pad(a.v.M);
            float* to = a.g.p + (store ? token : 0) * a.g.pitch;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int64_t v = v0 + 32 * i + 8 * q;
                    f16x4 h, l;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float g = __expf(acc[i][j][4 * q + e] - lse) - smooth;
                        if (at == 32 * i + 8 * q + e) g -= 1.f - a.v.ls;
                        g = valid && v + e < a.words ? g : 0.f;
                        if (a.part_db) db[16 * i + 4 * q + e] += g * row_scale;
                        _Float16 hi, lo;
                        split_value(g * kGScale, hi, lo);
                        h[e] = hi;
                        l[e] = lo;
                    }
                    if (store && v < a.g.pitch) { // 8 bytes of the group's h, and of its l: this half's four words
                        char* group = (char*)(to + (v - 4 * half));
                        *(f16x4*)(group + 8 * half) = h;
                        *(f16x4*)(group + 16 + 8 * half) = l;
                    }
                }
        }
        if (a.part_db) { // 64 values in each of 32 lanes, summed over the lanes: lane x keeps the sums of values 2 x and 2 x + 1 in bit-reversed order
#pragma unroll
            for (int step = 16, n = 32; step > 0; step >>= 1, n >>= 1) {
                const bool up = lane & step;
#pragma unroll
                for (int x = 0; x < n; ++x) {
                    const float give = up ? db[x] : db[x + n], keep = up ? db[x + n] : db[x];
                    db[x] = keep + __shfl_xor(give, step, 64);
                }
            }
            // after the steps this lane holds x = 32 b4 + 16 b3 + 8 b2 + 4 b1 + 2 b0 + {0, 1} with b the bits of its number
            const int x0 = 2 * (lane & 31);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int x = x0 + e, i = x >> 4, q = (x >> 2) & 3;
                const int64_t v = v0 + 32 * i + 8 * q + (x & 3);
                if (v < a.words) a.part_db[(2 * tn + (wave >> 1)) * a.v.V + a.first + v] = db[e];
            }
        }
    }
}

struct StoreArgs {
    float* c;
    int64_t rs, cs;
    const float* row_scale; // of C's rows, or NULL
    int accumulate;
};

template <bool A_KMAJOR, bool B_KMAJOR>
__global__ __launch_bounds__(256, 2) void vocab_product_kernel(const ProductArgs p, const StoreArgs s) {
    __shared__ __align__(1024) float lds[kStages * kStageBytes / 4];
    __shared__ uint32_t slots[2][4];
    int64_t tm, tn;
    tile_of(blockIdx.x, (uint32_t)p.tiles_m, (uint32_t)p.tiles_n, &tm, &tn);
    const int64_t m0 = tm * kTileM, n0 = tn * kTileN;
    f32x16 acc[4][2];
    split_tile<A_KMAJOR, B_KMAJOR>(acc, lds, p.a, m0, p.M, p.b, n0, p.N, p.k_steps);
    float inv = 1.f / (p.amax_a ? scale_from(p.amax_a, slots[0]) : kGScale);
    inv /= p.amax_b ? scale_from(p.amax_b, slots[1]) : kGScale;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t m = m0 + (wave & 1) * 128 + 32 * i + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
            if (m >= p.M) continue;
            const float scale = s.row_scale ? s.row_scale[m] * inv : inv;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t n = n0 + (wave >> 1) * 64 + 32 * j + (lane & 31);
                if (n >= p.N) continue;
                float* to = s.c + m * s.rs + n * s.cs;
                *to = s.accumulate ? *to + acc[i][j][e] * scale : acc[i][j][e] * scale;
            }
        }
}

// ---- rows ------------------------------------------------------------------------------------------------------------------------------

struct JoinArgs {
    VocabArgs v;
    const float2* part;
    const float *part_x, *target_logit;
    int64_t tiles;
    float *loss, *lse;
};

// 64 tokens a workgroup, the tiles of each dealt to the 4 wavefronts
__global__ __launch_bounds__(256) void vocab_join_kernel(const JoinArgs a) {
    __shared__ float s[3][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t token = (int64_t)blockIdx.x * 64 + lane, M = a.v.M;
    float top = -__builtin_inff(), sum = 0.f, sx = 0.f;
    if (token < M) {
        for (int64_t t = wave; t < a.tiles; t += 4) top = fmaxf(top, a.part[t * M + token].x);
        const float base = top == -__builtin_inff() ? 0.f : top;
        for (int64_t t = wave; t < a.tiles; t += 4) {
            const float2 p = a.part[t * M + token];
            sum += p.y * __expf(p.x - base);
            if (a.part_x) sx += a.part_x[t * M + token];
        }
    }
    s[0][wave][lane] = top; s[1][wave][lane] = sum; s[2][wave][lane] = sx;
    __syncthreads();
    if (wave || token >= M) return;
    top = fmaxf(fmaxf(s[0][0][lane], s[0][1][lane]), fmaxf(s[0][2][lane], s[0][3][lane]));
    const float base = top == -__builtin_inff() ? 0.f : top;
    sum = sx = 0.f;
    for (int w = 0; w < 4; ++w) sum += s[1][w][lane] * __expf(s[0][w][lane] - base), sx += s[2][w][lane];
    const float lse = base + logf(sum);
    a.lse[token] = lse;
    const int64_t t = target_of(a.v, token);
    float loss = 0.f;
    if (t != a.v.ignore) {
        if (t < 0 || t >= a.v.V) loss = __builtin_nanf("");
        else {
            loss = lse - a.target_logit[token];
            if (a.v.ls > 0.f) loss = (1.f - a.v.ls) * loss + a.v.ls * (lse - sx / (float)a.v.V);
        }
    }
    a.loss[token] = loss;
}

// The sum of the rows' losses (in 64 bits, a fixed order) and the number of rows that count: one workgroup.
__global__ __launch_bounds__(1024) void vocab_total_kernel(const VocabArgs v, const float* __restrict loss, float* loss_sum, int32_t* valid) {
    __shared__ double s[1024];
    __shared__ int c[1024];
    const int t = threadIdx.x;
    double sum = 0.0;
    int count = 0;
    for (int64_t m = t; m < v.M; m += 1024) {
        sum += loss[m];
        count += target_of(v, m) != v.ignore;
    }
    s[t] = sum;
    c[t] = count;
    for (int step = 512; step > 0; step >>= 1) {
        __syncthreads();
        if (t < step) s[t] += s[t + step], c[t] += c[t + step];
    }
    if (t == 0) *loss_sum = (float)s[0], *valid = c[0];
}

// scale_m: the factor of row m of the gradient
__global__ __launch_bounds__(256) void vocab_row_scale_kernel(const VocabArgs v, const float* upstream, int reduction, const int32_t* valid, float* scale) {
    const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (m >= v.M) return;
    float s = 0.f;
    if (target_of(v, m) != v.ignore) {
        s = upstream[reduction == 0 ? m : 0];
        if (reduction == 2) s /= (float)(*valid > 1 ? *valid : 1);
    }
    scale[m] = s;
}

__global__ __launch_bounds__(256) void vocab_db_kernel(const float* __restrict part, int64_t parts, int64_t V, float* db, int accumulate) {
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v >= V) return;
    float s = 0.f;
    for (int64_t i = 0; i < parts; ++i) s += part[i * V + v];
    db[v] = accumulate ? db[v] + s : s;
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------

struct Plan {
    SplitMatrix h, w, hs, g;
    uint32_t *amax_h, *amax_w, *amax_hs;
    float2* part;
    float *part_x, *target_logit, *row_scale, *part_db;
    int64_t piece; // words
};

int64_t tiles_of(int64_t n, int64_t t) { return (n + t - 1) / t; }

SplitMatrix take_split(Workspace& ws, int64_t rows, int64_t cols) {
    SplitMatrix m{nullptr, split_pad(cols), rows};
    m.p = ws.take<float>(split_pad(rows) * m.pitch);
    return m;
}

// W is split in the order in which it lies in memory, rows of words (a transposed embedding) or rows of D; both sizes fit either
void plan_operands(Workspace& ws, Plan& p, int64_t M, int64_t D, int64_t V, bool word_rows) {
    p.h = take_split(ws, M, D);
    p.w = SplitMatrix{ws.take<float>(split_pad(V) * split_pad(D)), word_rows ? split_pad(D) : split_pad(V), word_rows ? V : D};
    p.amax_h = ws.take<uint32_t>(kAmaxParts);
    p.amax_w = ws.take<uint32_t>(kAmaxParts);
}
void plan_forward(Workspace& ws, Plan& p, int64_t M, int64_t D, int64_t V, bool word_rows) {
    plan_operands(ws, p, M, D, V, word_rows);
    p.part = ws.take<float2>(tiles_of(V, kTileM) * M);
    p.part_x = ws.take<float>(tiles_of(V, kTileM) * M);
    p.target_logit = ws.take<float>(M);
}
void plan_backward(Workspace& ws, Plan& p, int64_t M, int64_t D, int64_t V, bool word_rows) {
    plan_operands(ws, p, M, D, V, word_rows);
    p.hs = take_split(ws, M, D);
    p.amax_hs = ws.take<uint32_t>(kAmaxParts);
    p.row_scale = ws.take<float>(M);
    p.part_db = ws.take<float>(2 * tiles_of(M, kTileN) * V);
    const int64_t most = std::max<int64_t>(kTileM, kPieceValues / split_pad(M) / kTileM * kTileM);
    p.piece = tiles_of(tiles_of(V, tiles_of(V, most)), kTileM) * kTileM; // pieces of equal size
    p.g = take_split(ws, M, std::min(p.piece, V));
}

int check_sizes(int64_t M, int64_t D, int64_t V, const char* who) {
    if (M < 0 || D < 1 || V < 1) return refuse(TENMO_ERR_INVALID_SHAPE, "%s: needs tokens >= 0, a dimension >= 1 and a vocabulary >= 1", who);
    if (M > 1 << 22 || D > 1 << 20 || V > 1 << 22) return refuse(TENMO_ERR_UNSUPPORTED, "%s: more than 2^22 tokens, 2^20 dimensions or 2^22 words", who);
    return 0;
}

int check_call(const tenmo_view* H, const tenmo_view* W, const float* bias, const void* target, int32_t is64, int64_t ignore, float ls, const char* who, VocabArgs* v) {
    if (int rc = check_operand(H, 2, 2, who, "H")) return rc;
    if (int rc = check_operand(W, 2, 2, who, "W")) return rc;
    if (W->shape[0] != H->shape[1]) return refuse(TENMO_ERR_INVALID_SHAPE, "%s: inner dims must match, got %lld and %lld", who, (long long)H->shape[1], (long long)W->shape[0]);
    if (int rc = check_sizes(H->shape[0], H->shape[1], W->shape[1], who)) return rc;
    if (!(ls >= 0.f && ls <= 1.f)) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: label_smoothing must be in [0, 1], got %g", who, (double)ls);
    *v = VocabArgs{H->shape[0], W->shape[1], H->shape[1], bias, target, is64 ? 1 : 0, ignore, ls};
    return 0;
}

Source source_h(const tenmo_view* H, const float* row_scale) { return Source{H->data + H->offset, H->shape[0], H->shape[1], H->strides[0], H->strides[1], row_scale}; }
bool rows_of_words(const tenmo_view* W) { return W->strides[0] == 1 && W->shape[0] > 1; }
Source source_w(const tenmo_view* W) {
    if (rows_of_words(W)) return Source{W->data + W->offset, W->shape[1], W->shape[0], W->strides[1], W->strides[0], nullptr};
    return Source{W->data + W->offset, W->shape[0], W->shape[1], W->strides[0], W->strides[1], nullptr};
}

void launch_split(const SplitJobs& j, int jobs, const LibraryState& lib) {
    int64_t groups = 0;
    for (int i = 0; i < jobs; ++i) groups = std::max(groups, split_pad(j.src[i].rows) * j.dst[i].pitch / 8);
    hipLaunchKernelGGL(vocab_amax_kernel, dim3(kAmaxParts, jobs), dim3(256), 0, lib.stream, j);
    hipLaunchKernelGGL(vocab_split_kernel, dim3((unsigned)std::min<int64_t>(tiles_of(groups, 256), 16 * lib.cus), jobs), dim3(256), 0, lib.stream, j);
}

ProductArgs product(const SplitMatrix& a, const uint32_t* amax_a, const SplitMatrix& b, const uint32_t* amax_b, int64_t M, int64_t N, int64_t K) {
    return ProductArgs{a, b, amax_a, amax_b, M, N, split_pad(K) / kStepK, tiles_of(M, kTileM), tiles_of(N, kTileN)};
}
dim3 grid_of(const ProductArgs& p) { return dim3((unsigned)(p.tiles_m * p.tiles_n)); }

// the words `first` .. of the split W
SplitMatrix words_of(const SplitMatrix& w, int64_t first, bool word_rows) { return SplitMatrix{w.p + (word_rows ? first * w.pitch : first), w.pitch, w.rows}; }

} // namespace
} // namespace tenmo

using namespace tenmo;

extern "C" {

int64_t tenmo_hip_vocabulary_loss_forward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocabulary) {
    if (int rc = check_sizes(tokens, dim, vocabulary, "tenmo_hip_vocabulary_loss_forward_workspace_bytes")) return rc;
    Workspace ws(nullptr, 0);
    Plan p{};
    if (tokens) plan_forward(ws, p, tokens, dim, vocabulary, true);
    return ws.used();
}

int tenmo_hip_vocabulary_loss_forward_f32(const tenmo_view* H, const tenmo_view* W, const float* bias, const void* target,
                                          int32_t target_is_int64, int64_t ignore_index, float label_smoothing,
                                          float* per_sample_loss, float* lse, float* loss_sum, int32_t* valid_count,
                                          void* workspace, int64_t workspace_bytes, int32_t sync) {
    const char* who = "tenmo_hip_vocabulary_loss_forward_f32";
    VocabArgs v{};
    if (int rc = check_call(H, W, bias, target, target_is_int64, ignore_index, label_smoothing, who, &v)) return rc;
    if (!loss_sum || !valid_count || (v.M > 0 && (!target || !per_sample_loss || !lse))) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    Call call(who);
    if (int rc = call.begin()) return rc;
    const hipStream_t stream = call.state.stream;
    if (v.M > 0) {
        const bool word_rows = rows_of_words(W);
        Workspace ws(workspace, workspace_bytes);
        Plan p{};
        plan_forward(ws, p, v.M, v.D, v.V, word_rows);
        if (int rc = ws.check(who)) return rc;
        SplitJobs j{};
        j.src[0] = source_w(W); j.amax[0] = p.amax_w; j.dst[0] = p.w;
        j.src[1] = source_h(H, nullptr); j.amax[1] = p.amax_h; j.dst[1] = p.h;
        launch_split(j, 2, call.state);
        const ProductArgs g = product(p.w, p.amax_w, p.h, p.amax_h, v.V, v.M, v.D);
        LogitArgs a{};
        a.v = v; a.words = v.V; a.part = p.part; a.part_x = label_smoothing > 0.f ? p.part_x : nullptr; a.target_logit = p.target_logit;
        if (word_rows) hipLaunchKernelGGL((vocab_logits_kernel<true, false>), grid_of(g), dim3(256), 0, stream, g, a);
        else hipLaunchKernelGGL((vocab_logits_kernel<false, false>), grid_of(g), dim3(256), 0, stream, g, a);
        const JoinArgs jn{v, p.part, a.part_x, p.target_logit, g.tiles_m, per_sample_loss, lse};
        hipLaunchKernelGGL(vocab_join_kernel, dim3((unsigned)tiles_of(v.M, 64)), dim3(256), 0, stream, jn);
    }
    hipLaunchKernelGGL(vocab_total_kernel, dim3(1), dim3(1024), 0, stream, v, per_sample_loss, loss_sum, valid_count);
    return call.finish(sync);
}

int64_t tenmo_hip_vocabulary_loss_backward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocabulary) {
    if (int rc = check_sizes(tokens, dim, vocabulary, "tenmo_hip_vocabulary_loss_backward_workspace_bytes")) return rc;
    Workspace ws(nullptr, 0);
    Plan p{};
    if (tokens) plan_backward(ws, p, tokens, dim, vocabulary, true);
    return ws.used();
}

int tenmo_hip_vocabulary_loss_backward_f32(const tenmo_view* H, const tenmo_view* W, const float* bias, const void* target,
                                           int32_t target_is_int64, int64_t ignore_index, float label_smoothing, const float* lse,
                                           const float* upstream, int32_t reduction, const int32_t* valid_count,
                                           float* grad_H, const tenmo_view* grad_W, float* grad_bias, int32_t accumulate,
                                           void* workspace, int64_t workspace_bytes, int32_t sync) {
    const char* who = "tenmo_hip_vocabulary_loss_backward_f32";
    VocabArgs v{};
    if (int rc = check_call(H, W, bias, target, target_is_int64, ignore_index, label_smoothing, who, &v)) return rc;
    if (reduction < 0 || reduction > 2) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: reduction must be 0 (none), 1 (sum) or 2 (mean)", who);
    if (grad_W) {
        if (int rc = check_operand(grad_W, 2, 2, who, "grad_W")) return rc;
        for (int d = 0; d < 2; ++d) {
            if (grad_W->shape[d] != W->shape[d])
                return refuse(TENMO_ERR_INVALID_SHAPE, "%s: axis %d of grad_W has %lld elements, %lld needed", who, d, (long long)grad_W->shape[d], (long long)W->shape[d]);
            if (grad_W->shape[d] > 1 && grad_W->strides[d] == 0) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: grad_W has a stride of 0: its elements share a place", who);
        }
    }
    if (v.M > 0 && (!target || !lse || !upstream)) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (v.M > 0 && reduction == 2 && !valid_count) return refuse(TENMO_ERR_INVALID_ARGUMENT, "%s: the mean needs valid_count", who);
    Call call(who);
    if (int rc = call.begin()) return rc;
    if (!grad_H && !grad_W && !grad_bias) return 0;
    const hipStream_t stream = call.state.stream;
    const int add = accumulate ? 1 : 0;
    // dW as [words][D] or [D][words]: the axis with unit stride across the lanes
    float* gw = grad_W ? const_cast<float*>(grad_W->data) + grad_W->offset : nullptr;
    const int64_t gw_d = grad_W ? grad_W->strides[0] : 0, gw_v = grad_W ? grad_W->strides[1] : 0;
    const bool word_rows = rows_of_words(W);
    Workspace ws(workspace, workspace_bytes);
    Plan p{};
    if (v.M > 0) plan_backward(ws, p, v.M, v.D, v.V, word_rows);
    if (int rc = ws.check(who)) return rc;
    if (v.M > 0) {
        hipLaunchKernelGGL(vocab_row_scale_kernel, dim3((unsigned)tiles_of(v.M, 256)), dim3(256), 0, stream, v, upstream, (int)reduction, valid_count, p.row_scale);
        SplitJobs j{};
        j.src[0] = source_w(W); j.amax[0] = p.amax_w; j.dst[0] = p.w;
        j.src[1] = source_h(H, nullptr); j.amax[1] = p.amax_h; j.dst[1] = p.h;
        launch_split(j, 2, call.state);
        j.src[0] = source_h(H, p.row_scale); j.amax[0] = p.amax_hs; j.dst[0] = p.hs;
        if (grad_W) launch_split(j, 1, call.state);
    }
    const int64_t piece = v.M > 0 ? p.piece : v.V;
    for (int64_t first = 0; first < v.V; first += piece) {
        const int64_t words = std::min(piece, v.V - first);
        SplitMatrix G = p.g;
        G.pitch = split_pad(words);
        if (v.M > 0) {
            const SplitMatrix w = words_of(p.w, first, word_rows);
            const ProductArgs g = product(w, p.amax_w, p.h, p.amax_h, words, v.M, v.D);
            LogitArgs a{};
            a.v = v; a.first = first; a.words = words; a.lse = lse; a.row_scale = p.row_scale; a.g = G; a.part_db = grad_bias ? p.part_db : nullptr;
            if (word_rows) hipLaunchKernelGGL((vocab_logits_kernel<true, true>), grid_of(g), dim3(256), 0, stream, g, a);
            else hipLaunchKernelGGL((vocab_logits_kernel<false, true>), grid_of(g), dim3(256), 0, stream, g, a);
            if (grad_H) {
                const ProductArgs d = product(G, nullptr, w, p.amax_w, v.M, v.D, words);
                const StoreArgs s{grad_H, v.D, 1, p.row_scale, first > 0 || add};
                if (word_rows) hipLaunchKernelGGL((vocab_product_kernel<true, false>), grid_of(d), dim3(256), 0, stream, d, s);
                else hipLaunchKernelGGL((vocab_product_kernel<true, true>), grid_of(d), dim3(256), 0, stream, d, s);
            }
        }
        if (grad_W) {
            float* to = gw + first * gw_v;
            if (gw_d == 1 || gw_v != 1) {
                const ProductArgs d = product(G, nullptr, p.hs, p.amax_hs, words, v.D, v.M);
                hipLaunchKernelGGL((vocab_product_kernel<false, false>), grid_of(d), dim3(256), 0, stream, d, (StoreArgs{to, gw_v, gw_d, nullptr, add}));
            } else {
                const ProductArgs d = product(p.hs, p.amax_hs, G, nullptr, v.D, words, v.M);
                hipLaunchKernelGGL((vocab_product_kernel<false, false>), grid_of(d), dim3(256), 0, stream, d, (StoreArgs{to, gw_d, gw_v, nullptr, add}));
            }
        }
    }
    if (grad_bias) hipLaunchKernelGGL(vocab_db_kernel, dim3((unsigned)tiles_of(v.V, 256)), dim3(256), 0, stream, p.part_db, v.M > 0 ? 2 * tiles_of(v.M, kTileN) : 0, v.V, grad_bias, add);
    return call.finish(sync);
}

} // extern "C"
