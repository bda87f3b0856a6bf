// Cross-entropy of the logits x = H W + bias over a vocabulary, from the hidden states (include/tenmo_hip_transformer.h).
//
//   lse = log sum_v exp(x_v),  loss = (1 - ls) (lse - x_t) + ls (lse - mean_v x_v)
//   G = (exp(x - lse) - (1 - ls) [v = t] - ls / V) [t valid],  scale_m = the upstream gradient of row m
//   dH = scale (G W^T),  dW = (scale H)^T G,  db = sum_m scale_m G
//
// Bound: the matrix units, 2 M V D flop forward, 6 M V D backward (the logits again, dH, dW).  All three products run as split fp16 products
// (split_gemm.hpp); for few tokens or a small W, where reading W or latency is the bound, the kernels of vocabulary_few.hip take their place.
//   * forward: tiles of 256 words x 128 tokens; the words of a token lie in the registers of two lanes, so that a tile's maximum and sum of a token take
//     one exchange, and 8 bytes a token and tile leave the chip instead of 1 KiB of logits.  A second launch joins the tiles of a token in a fixed order.
//   * backward: a piece of the vocabulary at a time; the tiles of the first launch end as G in split form, which the next one multiplies with W and with H.  The piece is as large as 1 GiB of G allows.
//     Two forms of G, since its two products sum over different axes:
//       G W^T    G at 2^14.  A row is a token's, whose target has p - 1, itself right to 2^-24 of 1; the halves hold the others to 2^-40 of 1.
//       G^T H    scale_m G / (the scale of H's row m), which is what a word's row of dW is summed from: with a scale for each word and 64 tokens, a power of 2^6 that brings their largest into
//                2^8 .. 2^14 (split_gemm.hpp brings them to the word's smallest).  Words without a target have probabilities alone in their rows, however small, and tokens lie far apart in
//                their upstream gradients: at 2^14 for all, rows of words whose logits lie 16 below the others' were off by 5e-2 of what enters them, 20 below by 1 (700 tokens,
//                130 x 9000).  It costs a second G in memory and the scales, 1032 -> 1200 us, and factors as it is read, 1892 -> 1990 us (half of 8192 x 50257, D = 768).
#include "split_gemm.hpp"
#include "vocabulary.hpp"

#include <algorithm>
#include <type_traits>

namespace tenmo {
namespace {

constexpr float kGScale = 16384.f;
constexpr int kWordBits = 13, kMostClass = 18; // a word's scale: 2^(kWordBits + kCodeBits * class)
constexpr int64_t kPieceValues = 256 << 20; // of G, 4 bytes each

struct Source { // an operand in the order in which it is split: rows x cols
    const float* p;
    int64_t rows, cols, rs, cs;
};

// ---- amax and split -------------------------------------------------------------------------------------------------------------

// W has one scale, since it is summed over along either axis: its largest value first, then the halves.  H has a scale of its own in each row, so that no row loses anything to another (a row is
// one column of the logits' product; in G^T H the scales go into G); its halves come with the first launch.
struct SplitArgs {
    VocabArgs v;
    Upstream up;      // p NULL: forward
    Source w, h;
    uint32_t* amax_w; // kAmaxParts partial maxima
    uint32_t* top_f;  // backward, as many partial maxima: (kNoFactor + log2 of a token's factor over its scale of H) << kFactorShift, 0 without a token that counts
    SplitMatrix to_w, to_h;
    float* h_inverse; // [M]: 1 / the scale of a row of H
};
enum { kSplitW, kSplitH }; // blockIdx.y
constexpr int kNoFactor = 512, kFactorShift = 21; // (as bits of a normal float: the maxima are taken of those)
__device__ __forceinline__ int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }

__device__ __forceinline__ void split8(const float* x, float scale, float* to) {
    f16x8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        _Float16 hi, lo;
        split_value(x[e] * scale, hi, lo);
        h[e] = hi;
        l[e] = lo;
    }
    *(f16x8*)to = h;
    *(f16x8*)(to + 4) = l;
}
// columns c .. c + 7 of a row, zero behind the last
__device__ __forceinline__ void load8(float (&x)[8], const float* p, int64_t cs, int64_t c, int64_t cols) {
    if (cs == 1 && c + 7 < cols) {
        const f32x4 a = *(const f32x4_u*)(p + c), b = *(const f32x4_u*)(p + c + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = c + e < cols ? p[(c + e) * cs] : 0.f;
    }
}

// a wavefront a row
__device__ __forceinline__ void split_h_rows(const SplitArgs& a) {
    __shared__ uint32_t tops[4];
    const int lane = threadIdx.x & 63;
    uint32_t top_f = 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < split_pad(a.h.rows); r += 4 * kAmaxParts) {
        const float factor = r >= a.h.rows ? 0.f : a.up.p ? row_factor(a.v, a.up, r) : 1.f;
        const bool in = factor != 0.f; // rows without a part in the gradient are zeros, whatever they hold
        const float* p = a.h.p + (in ? r : 0) * a.h.rs;
        const int64_t cols = in ? a.h.cols : 0;
        uint32_t top = 0;
        float x[8];
        for (int64_t c = lane * 8; c < a.to_h.pitch; c += 512) {
            load8(x, p, a.h.cs, c, cols);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, finite_magnitude(x[e]));
        }
        top = wave_max_bits(top);
        const float scale = top ? split_scale(top) : 0x1p126f; // (a row of zeros has the smallest part in G^T H: it leaves the scales of the tokens beside it as they are)
        for (int64_t c = lane * 8; c < a.to_h.pitch; c += 512) {
            load8(x, p, a.h.cs, c, cols);
            split8(x, scale, a.to_h.p + r * a.to_h.pitch + c);
        }
        if (r < a.h.rows && lane == 0) a.h_inverse[r] = 1.f / scale;
        if (in && finite_magnitude(factor)) top_f = max(top_f, (uint32_t)(kNoFactor + exponent_of(factor) - exponent_of(scale)) << kFactorShift);
    }
    if (!a.top_f) return;
    if (lane == 0) tops[threadIdx.x >> 6] = top_f;
    __syncthreads();
    if (threadIdx.x == 0) a.top_f[blockIdx.x] = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
}

// four rows at a time: four loads in flight a thread
__global__ __launch_bounds__(256) void vocab_amax_kernel(const SplitArgs a) {
    __shared__ uint32_t slots[4];
    if (blockIdx.y == kSplitH) return split_h_rows(a);
    const Source& s = a.w;
    uint32_t top = 0;
    for (int64_t r0 = blockIdx.x; r0 < s.rows; r0 += 4 * kAmaxParts) {
        const float* p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = s.p + (r0 + u * kAmaxParts < s.rows ? r0 + u * kAmaxParts : s.rows - 1) * s.rs; // (the last row again where there is none)
        int64_t c = threadIdx.x * 4;
        if (s.cs == 1)
            for (; c + 3 < s.cols; c += 1024) {
                f32x4 x[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) x[u] = *(const f32x4_u*)(p[u] + c);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = max(top, finite_magnitude(x[u][e]));
            }
        for (; c < s.cols; c += 1024)
            for (int e = 0; e < 4 && c + e < s.cols; ++e)
#pragma unroll
                for (int u = 0; u < 4; ++u) top = max(top, finite_magnitude(p[u][(c + e) * s.cs]));
    }
    top = wave_max_bits(top);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) a.amax_w[blockIdx.x] = max(max(slots[0], slots[1]), max(slots[2], slots[3]));
}

// the largest of the partial maxima, in every thread of a workgroup of 256
__device__ __forceinline__ uint32_t top_from(const uint32_t* __restrict amax, uint32_t* slots) {
    uint32_t top = 0;
    for (int i = threadIdx.x; i < kAmaxParts; i += 256) top = max(top, amax[i]);
    top = wave_max_bits(top);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = top;
    __syncthreads();
    return max(max(slots[0], slots[1]), max(slots[2], slots[3]));
}
__device__ __forceinline__ float scale_from(const uint32_t* __restrict amax, uint32_t* slots) { return split_scale(top_from(amax, slots)); }
// log2 of the largest of the tokens' factors over their scales of H, rounded down
__device__ __forceinline__ int factor_from(const uint32_t* __restrict top_f, uint32_t* slots) { return (int)(top_from(top_f, slots) >> kFactorShift) - kNoFactor; }

__global__ __launch_bounds__(256) void vocab_split_kernel(const SplitArgs a) {
    __shared__ uint32_t slots[4];
    const Source& s = a.w;
    const int64_t pitch = a.to_w.pitch;
    const float scale = scale_from(a.amax_w, slots);
    const int64_t groups = pitch / 8, all = split_pad(s.rows) * groups;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / groups, c = (i - r * groups) * 8;
        float x[8];
        load8(x, s.p + (r < s.rows ? r : 0) * s.rs, s.cs, c, r < s.rows ? s.cols : 0);
        split8(x, scale, a.to_w.p + r * pitch + c);
    }
}

// ---- the products --------------------------------------------------------------------------------------------------------------------

struct ProductArgs {
    SplitMatrix a, b;
    const uint32_t *amax_a, *amax_b; // NULL: G, whose scale is kGScale
    int64_t M, N, k_steps;
    int64_t tiles_m, tiles_n;
    int64_t run_steps, run_stride; // K steps of a run, and floats from one run's result to the next
    // G with a scale for each word
    Codes codes;
    const int* unit;       // [words]: log2 of the scale that the codes bring it to
    const uint32_t* top_f; // SplitArgs
};

struct LogitArgs {
    VocabArgs v;
    int64_t first; // word of the piece's first row
    int64_t words; // of the piece
    const float* h_inverse;
    // forward
    float2* part;      // [tile][token]: maximum and sum
    float* part_x;     // [tile][token]: sum of the logits, with label smoothing
    float* target_logit; // [token]
    // backward
    const float* lse;
    Upstream up;
    SplitMatrix g, gw; // for dH, and for dW; p NULL: not wanted
    uint8_t* word_class; // [blocks of 64 tokens][gw.pitch]
    const uint32_t* top_f; // SplitArgs
    float* part_db; // [2 * token tiles][V], with a wanted bias gradient
};

// A token's 4 words in this lane, and 4 in the lane 32 further, in split form: the two lanes hold half each of a group of eight; the lower one stores the eight h, the upper one the eight l
__device__ __forceinline__ f32x4 split_words(f32x4 x, float one) {
    union { f16x4 v[2]; uint32_t u[4]; f32x4 f; } y;
    asm("" : "+v"(x)); // (a product: one rounding of it for both halves)
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[0][e] = (_Float16)x[e];
    asm("" : "+v"(y.v[0]));
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[1][e] = (_Float16)__builtin_fmaf(x[e], one, -(float)y.v[0][e]);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const auto z = __builtin_amdgcn_permlane32_swap(y.u[w], y.u[2 + w], false, false);
        y.u[w] = z[0];
        y.u[2 + w] = z[1];
    }
    return y.f;
}

// The scales of a wavefront's 16 words from their magnitudes in this lane, the same in the 32 lanes of a half, and their classes to memory (four words of the half at `classes` + 8 q)
template <int CTRL>
__device__ __forceinline__ uint32_t lane_move_bits(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ void word_scales(float (&x)[16], uint8_t* classes, int lane, int words) {
    uint32_t cls[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { // the lower 16 lanes of a half go on with words 0 .. 7, the upper with 8 .. 15
        const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[e]), __float_as_uint(x[e + 8]), false, false);
        uint32_t top = max(y[0], y[1]); // (magnitudes: ordered as their bits are)
        top = max(top, (uint32_t)lane_move_bits<0xB1>(top));
        top = max(top, (uint32_t)lane_move_bits<0x4E>(top));
        top = max(top, (uint32_t)lane_move_bits<0x141>(top));
        top = max(top, (uint32_t)lane_move_bits<0x140>(top));
        const int below = 127 - (int)(top >> 23); // top in [2^-below, 2^(1 - below))
        const uint32_t c = (uint32_t)(fmaxf((float)below, 0.f) * (342.f / 2048.f)); // / kCodeBits, exactly so
        cls[e] = c < kMostClass ? c : kMostClass;
        const uint32_t scale = (127 + kWordBits + __umul24(cls[e], kCodeBits)) << 23;
        const auto z = __builtin_amdgcn_permlane16_swap(scale, scale, false, false);
        x[e] = __uint_as_float(z[0]);
        x[e + 8] = __uint_as_float(z[1]);
    }
    if ((lane & 15) == 0) {
        const int q = (lane >> 4) & 1; // groups 2 q and 2 q + 1
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (8 * (2 * q + u) < words) *(uint32_t*)(classes + 8 * (2 * q + u)) = cls[4 * u] | cls[4 * u + 1] << 8 | cls[4 * u + 2] << 16 | cls[4 * u + 3] << 24;
    }
}

template <bool A_KMAJOR, bool GRAD>
__global__ __launch_bounds__(256, 2) void vocab_logits_kernel(const ProductArgs p, const LogitArgs a) {
    __shared__ __align__(1024) float lds[kStages * kStageBytes / 4];
    __shared__ uint32_t slots[4];
    int64_t tm, tn;
    tile_of(blockIdx.x, (uint32_t)p.tiles_m, (uint32_t)p.tiles_n, &tm, &tn);
    const int64_t m0 = tm * kTileM, n0 = tn * kTileN;
    f32x16 acc[4][2];
    split_tile<A_KMAJOR, true>(acc, lds, p.a, m0, p.M, p.b, n0, p.N, 0, p.k_steps);
    const float inv_w = 1.f / scale_from(p.amax_a, slots);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int64_t v0 = m0 + (wave & 1) * 128 + 4 * half; // of the piece; register e of block i is v0 + 32 i + 8 (e / 4) + e % 4
    // logits in place
    float inv[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t token = n0 + (wave >> 1) * 64 + 32 * j + (lane & 31);
        inv[j] = a.h_inverse[token < a.v.M ? token : a.v.M - 1]; // (applied after inv_w: the product of the two may be out of range)
    }
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
                for (int j = 0; j < 2; ++j) acc[i][j][4 * q + e] = acc[i][j][4 * q + e] * inv_w * inv[j] + bias[e];
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
        const float smooth = a.v.ls / (float)a.v.V, one = variable_one();
        __shared__ uint32_t slots_f[4];
        const int top_f = a.gw.p ? factor_from(a.top_f, slots_f) : 0;
        bool valid[2], store[2];
        float lse[2], row_scale[2], factor[2];
        int at[2]; // the target's place in this lane's words
        float *to_g[2], *to_gw[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t token = n0 + (wave >> 1) * 64 + 32 * j + (lane & 31);
            row_scale[j] = token < a.v.M ? row_factor(a.v, a.up, token) : 0.f;
            valid[j] = row_scale[j] != 0.f;
            lse[j] = valid[j] ? a.lse[token] : 0.f;
            factor[j] = __builtin_amdgcn_ldexpf(row_scale[j], exponent_of(inv[j]) - top_f); // below 2
            const int64_t place = valid[j] ? target_of(a.v, token) - a.first - v0 : -1;
            at[j] = place >= 0 && place < 128 ? (int)place : -1;
            store[j] = token < split_pad(a.v.M);
            to_g[j] = a.g.p + (store[j] ? token : 0) * a.g.pitch + v0;
            to_gw[j] = a.gw.p + (store[j] ? token : 0) * a.gw.pitch + v0;
        }
        const bool here = __any(at[0] >= 0 || at[1] >= 0); // a target among this wavefront's words: one in three at 50257 words
        const int words = (int)(a.words - v0 < 256 ? a.words - v0 : 256), pitch = (int)((a.g.p ? a.g.pitch : a.gw.pitch) - v0 < 256 ? (a.g.p ? a.g.pitch : a.gw.pitch) - v0 : 256);
        uint8_t* const classes = a.word_class + ((n0 >> 6) + (wave >> 1)) * a.gw.pitch + v0;
        // WHOLE: every word and token of the tile is there
        auto end = [&](auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int w = 32 * i + 8 * (e >> 2) + (e & 3);
                        const float g = __expf(acc[i][j][e] - lse[j]) - smooth;
                        acc[i][j][e] = valid[j] && (WHOLE || w < words) ? g : 0.f;
                    }
                if (here)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            acc[i][j][e] -= at[j] == 32 * i + 8 * (e >> 2) + (e & 3) ? 1.f - a.v.ls : 0.f;
                if (a.part_db) { // 16 values in each of 32 lanes, summed over the lanes: lanes 2 x and 2 x + 1 end with the sum of the value whose number has x's bits
                    float db[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) db[e] = acc[i][0][e] * row_scale[0] + acc[i][1][e] * row_scale[1];
#pragma unroll
                    for (int step = 16, n = 8; step > 1; step >>= 1, n >>= 1) {
                        const bool up = lane & step;
#pragma unroll
                        for (int x = 0; x < n; ++x) {
                            const float give = up ? db[x] : db[x + n], keep = up ? db[x + n] : db[x];
                            db[x] = keep + __shfl_xor(give, step, 64);
                        }
                    }
                    db[0] += __shfl_xor(db[0], 1, 64);
                    const int x = (lane & 31) >> 1;
                    const int64_t v = v0 + 32 * i + 8 * (x >> 2) + (x & 3);
                    if (!(lane & 1) && v < a.words) a.part_db[(2 * tn + (wave >> 1)) * a.v.V + a.first + v] = db[0];
                }
                if (a.g.p)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            f32x4 x;
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = acc[i][j][4 * q + e] * kGScale;
                            x = split_words(x, one);
                            if (WHOLE || (store[j] && 32 * i + 8 * q < pitch)) *(f32x4*)(to_g[j] + 32 * i + 8 * q) = x;
                        }
                if (!a.gw.p) continue;
                float scale[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    acc[i][0][e] *= factor[0];
                    acc[i][1][e] *= factor[1];
                    scale[e] = fmaxf(fabsf(acc[i][0][e]), fabsf(acc[i][1][e]));
                }
                word_scales(scale, classes + 32 * i, lane, pitch - 32 * i);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f32x4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = acc[i][j][4 * q + e] * scale[4 * q + e];
                        x = split_words(x, one);
                        if (WHOLE || (store[j] && 32 * i + 8 * q < pitch)) *(f32x4*)(to_gw[j] + 32 * i + 8 * q) = x;
                    }
            }
        };
        if (!edge && n0 + kTileN <= a.v.M) end(std::true_type{});
        else end(std::false_type{});
    }
}

struct StoreArgs {
    float* c;
    int64_t rs, cs;
    int accumulate;
};

template <bool A_KMAJOR, bool B_KMAJOR, int CODED>
__device__ __forceinline__ void product_tile(const ProductArgs& p, const StoreArgs& s, uint32_t id, float* lds, uint32_t (*slots)[4]) {
    int64_t tm, tn;
    const uint32_t tiles = (uint32_t)(p.tiles_m * p.tiles_n), run = id / tiles;
    tile_of(id - run * tiles, (uint32_t)p.tiles_m, (uint32_t)p.tiles_n, &tm, &tn);
    const int64_t m0 = tm * kTileM, n0 = tn * kTileN;
    const int64_t k0 = __builtin_amdgcn_readfirstlane((uint32_t)(run * p.run_steps));
    const int64_t steps = p.k_steps - k0 < p.run_steps ? p.k_steps - k0 : p.run_steps;
    f32x16 acc[4][2];
    split_tile<A_KMAJOR, B_KMAJOR, CODED>(acc, lds, p.a, m0, p.M, p.b, n0, p.N, k0, steps, p.codes);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if constexpr (CODED == kPlain) {
        const float inv = 1.f / kGScale / scale_from(p.amax_b, slots[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] *= inv;
    } else { // each word's scale, and the tokens' largest factor
        const int top_f = factor_from(p.top_f, slots[0]);
        if constexpr (CODED == kCodedA) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int up = top_f - p.unit[m0 + (wave & 1) * 128 + 32 * i + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)];
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j][e] = __builtin_amdgcn_ldexpf(acc[i][j][e], up);
                }
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int up = top_f - p.unit[n0 + (wave >> 1) * 64 + 32 * j + (lane & 31)];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_amdgcn_ldexpf(acc[i][j][e], up);
            }
        }
    }
    float* c = s.c + (int64_t)run * p.run_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t m = m0 + (wave & 1) * 128 + 32 * i + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
            if (m >= p.M) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t n = n0 + (wave >> 1) * 64 + 32 * j + (lane & 31);
                if (n >= p.N) continue;
                float* to = c + m * s.rs + n * s.cs;
                *to = s.accumulate ? *to + acc[i][j][e] : acc[i][j][e];
            }
        }
}

// Both products of a piece in one launch, since neither fills the chip evenly by itself: the first `h_tiles` workgroups are G W^T (its reduction over the words cut into runs of about the
// length of the other's, each into a sum of its own), the others G^T H (words in the rows), or its transpose.
template <bool W_KMAJOR, bool WORD_ROWS>
__global__ __launch_bounds__(256, 2) void vocab_products_kernel(const ProductArgs h, const StoreArgs sh, uint32_t h_tiles, const ProductArgs w, const StoreArgs sw) {
    __shared__ __align__(1024) float lds[kStages * kStageBytes / 4];
    __shared__ uint32_t slots[2][4];
    if (blockIdx.x < h_tiles) product_tile<true, W_KMAJOR, kPlain>(h, sh, blockIdx.x, lds, slots);
    else product_tile<false, false, WORD_ROWS ? kCodedA : kCodedB>(w, sw, blockIdx.x - h_tiles, lds, slots);
}

// Each word's scale in G^T H, the smallest of those of its blocks of 64 tokens, and what brings the others to it
__global__ __launch_bounds__(256) void vocab_unit_kernel(const uint8_t* __restrict classes, int64_t pitch, int64_t blocks, uint32_t* __restrict codes, int* __restrict unit) {
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v >= pitch) return;
    uint32_t least = kMostClass;
#pragma unroll 16
    for (int64_t t = 0; t < blocks; ++t) least = min(least, (uint32_t)classes[t * pitch + v]);
    unit[v] = kWordBits + kCodeBits * (int)least;
    for (int64_t t = 0; t < blocks; t += kCodesAWord) {
        uint32_t word = 0;
#pragma unroll
        for (int u = 0; u < kCodesAWord; ++u) word |= min((t + u < blocks ? classes[(t + u) * pitch + v] : least) - least, (uint32_t)kMostCode) << (4 * u);
        codes[t / kCodesAWord * pitch + v] = word;
    }
}

// ---- rows ------------------------------------------------------------------------------------------------------------------------------

struct JoinArgs {
    VocabArgs v;
    const float2* part;
    const float *part_x, *target_logit;
    int64_t tiles;
    float *loss, *lse;
    float* loss_sum; // with one workgroup: the sum of the losses as well, and the tokens that count
    int32_t* valid_count;
};

// 64 tokens a workgroup, the tiles of each dealt to the 16 wavefronts
__global__ __launch_bounds__(1024) void vocab_join_kernel(const JoinArgs a) {
    __shared__ float s[3][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t token = (int64_t)blockIdx.x * 64 + lane, M = a.v.M;
    float top = -__builtin_inff(), sum = 0.f, sx = 0.f;
    constexpr int U = 8; // tiles in flight a thread (the last one again where there is none)
    if (token < M)
        for (int64_t t0 = wave; t0 < a.tiles; t0 += 16 * U) {
            float2 p[U];
            float x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t t = t0 + 16 * u < a.tiles ? t0 + 16 * u : a.tiles - 1;
                p[u] = a.part[t * M + token];
                x[u] = a.part_x ? a.part_x[t * M + token] : 0.f;
            }
            float now = top;
#pragma unroll
            for (int u = 0; u < U; ++u) now = fmaxf(now, p[u].x);
            const float base = now == -__builtin_inff() ? 0.f : now;
            sum *= __expf(top - base);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = t0 + 16 * u < a.tiles;
                sum += in ? p[u].y * __expf(p[u].x - base) : 0.f;
                sx += in ? x[u] : 0.f;
            }
            top = now;
        }
    s[0][wave][lane] = top; s[1][wave][lane] = sum; s[2][wave][lane] = sx;
    __syncthreads();
    if (wave) return;
    float loss = 0.f;
    bool counts = false;
    if (token < M) {
        for (int w = 1; w < 16; ++w) top = fmaxf(top, s[0][w][lane]);
        const float base = top == -__builtin_inff() ? 0.f : top;
        sum = sx = 0.f;
        for (int w = 0; w < 16; ++w) sum += s[1][w][lane] * __expf(s[0][w][lane] - base), sx += s[2][w][lane];
        const float lse = base + logf(sum);
        a.lse[token] = lse;
        const int64_t t = target_of(a.v, token);
        counts = t != a.v.ignore;
        if (counts) {
            if (t < 0 || t >= a.v.V) loss = __builtin_nanf("");
            else {
                loss = lse - a.target_logit[token];
                if (a.v.ls > 0.f) loss = (1.f - a.v.ls) * loss + a.v.ls * (lse - sx / (float)a.v.V);
            }
        }
        a.loss[token] = loss;
    }
    if (!a.loss_sum) return;
    double total = loss;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d, 64);
    const int many = __popcll(__ballot(counts));
    if (lane == 0) *a.loss_sum = (float)total, *a.valid_count = many;
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

// dH: the runs' sums added in order, times each row's factor
__global__ __launch_bounds__(256) void vocab_dh_kernel(const float* __restrict part, int64_t runs, const VocabArgs v, const Upstream up, float* __restrict dh, int accumulate) {
    const int64_t D = v.D, all = v.M * D;
    for (int64_t x = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; x < all; x += (int64_t)gridDim.x * 1024) {
        if (x + 3 < all) {
            f32x4 s = *(const f32x4*)(part + x);
#pragma unroll 16
            for (int64_t r = 1; r < runs; ++r) s += *(const f32x4_u*)(part + r * all + x);
            const int64_t m = x / D;
            const float factor = row_factor(v, up, m);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] *= x + e < (m + 1) * D ? factor : row_factor(v, up, (x + e) / D);
            if (accumulate) s += *(const f32x4_u*)(dh + x);
            *(f32x4_u*)(dh + x) = s;
        } else {
            for (int64_t y = x; y < all; ++y) {
                float s = part[y];
                for (int64_t r = 1; r < runs; ++r) s += part[r * all + y];
                s *= row_factor(v, up, y / D);
                dh[y] = accumulate ? dh[y] + s : s;
            }
        }
    }
}

// dW of a piece: the runs' sums [rows][cols] added in order (zeros without a run)
__global__ __launch_bounds__(256) void vocab_dw_kernel(const float* __restrict part, int64_t runs, int64_t rows, int64_t cols, const StoreArgs s) {
    const int64_t all = rows * cols;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < all; x += (int64_t)gridDim.x * 256) {
        float sum = runs > 0 ? part[x] : 0.f;
#pragma unroll 8
        for (int64_t r = 1; r < runs; ++r) sum += part[r * all + x];
        float* to = s.c + x / cols * s.rs + x % cols * s.cs;
        *to = s.accumulate ? *to + sum : sum;
    }
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
    SplitMatrix h, w, g, gw;
    uint32_t *amax_w, *top_f, *codes;
    uint8_t* word_class;
    int* unit;
    float* h_inverse;
    float2* part;
    float *part_x, *target_logit, *part_db, *part_h, *part_w;
    int64_t piece;  // words
    int64_t runs;   // of the words of a piece, in G W^T
    int64_t w_runs; // of the tokens, in G^T H
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
    p.h_inverse = ws.take<float>(M);
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
    p.top_f = ws.take<uint32_t>(kAmaxParts);
    p.part_db = ws.take<float>(2 * tiles_of(M, kTileN) * V);
    const int64_t most = std::max<int64_t>(kTileM, kPieceValues / split_pad(M) / kTileM * kTileM);
    p.piece = tiles_of(tiles_of(V, tiles_of(V, most)), kTileM) * kTileM; // pieces of equal size
    p.piece = std::min(p.piece, split_pad(V));
    p.g = take_split(ws, M, p.piece);
    p.gw = take_split(ws, M, p.piece);
    p.word_class = ws.take<uint8_t>(2 * tiles_of(M, kTileN) * p.gw.pitch);
    p.codes = ws.take<uint32_t>(tiles_of(tiles_of(M, kCodeK), kCodesAWord) * p.gw.pitch);
    p.unit = ws.take<int>(tiles_of(p.piece, kTileM) * kTileM); // (a tile reads those of all its rows)
    // As many runs as bring their length near the other product's (but not below 2048), or as fill two workgroups a CU where there are fewer
    // tiles than that, none shorter than 128 words.
    const int64_t tiles = tiles_of(M, kTileM) * tiles_of(D, kTileN);
    p.runs = std::max<int64_t>(1, std::max(p.piece / std::max<int64_t>(M, 2048), std::min(p.piece / 128, 512 / tiles)));
    p.part_h = ws.take<float>(p.runs * M * D);
    // The same of the tokens where the weight's gradient has few tiles (128 x 300, 16384 tokens: 92 us backward, 667 with one run)
    p.w_runs = std::max<int64_t>(1, std::min(M / 128, 512 / (tiles_of(p.piece, kTileM) * tiles_of(D, kTileN))));
    if (p.w_runs > 1) p.part_w = ws.take<float>(p.w_runs * p.piece * D);
}

int check_sizes(int64_t M, int64_t D, int64_t V, const char* who) {
    if (M < 0 || D < 1 || V < 1) return refuse(TENMO_ERR_INVALID_SHAPE, "%s: needs tokens >= 0, a dimension >= 1 and a vocabulary >= 1", who);
    const int64_t most = (int64_t)1 << 38; // a launch holds 2^32 threads: 2^24 tiles of 2^15 values
    if (M > 1 << 22 || D > 1 << 20 || V > 1 << 22 || M * V > most || D * V > most || M * D > most)
        return refuse(TENMO_ERR_UNSUPPORTED, "%s: more than 2^22 tokens, 2^20 dimensions, 2^22 words or 2^38 values of a matrix", who);
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

Source source_h(const tenmo_view* H) { return Source{H->data + H->offset, H->shape[0], H->shape[1], H->strides[0], H->strides[1]}; }
Operand2 operand(const tenmo_view* x) { return Operand2{x->data + x->offset, x->strides[0], x->strides[1]}; }
bool rows_of_words(const tenmo_view* W) { return W->strides[0] == 1 && W->shape[0] > 1; }
Source source_w(const tenmo_view* W) {
    if (rows_of_words(W)) return Source{W->data + W->offset, W->shape[1], W->shape[0], W->strides[1], W->strides[0]};
    return Source{W->data + W->offset, W->shape[0], W->shape[1], W->strides[0], W->strides[1]};
}

// W and H
void launch_split(const Plan& p, const tenmo_view* H, const tenmo_view* W, const VocabArgs& v, const Upstream& up, const LibraryState& lib) {
    const SplitArgs a{v, up, source_w(W), source_h(H), p.amax_w, p.top_f, p.w, p.h, p.h_inverse};
    const int64_t groups = split_pad(a.w.rows) * p.w.pitch / 8;
    hipLaunchKernelGGL(vocab_amax_kernel, dim3(kAmaxParts, 2), dim3(256), 0, lib.stream, a);
    hipLaunchKernelGGL(vocab_split_kernel, dim3((unsigned)std::min<int64_t>(tiles_of(groups, 256), 16 * lib.cus)), dim3(256), 0, lib.stream, a);
}

ProductArgs product(const SplitMatrix& a, const uint32_t* amax_a, const SplitMatrix& b, const uint32_t* amax_b, int64_t M, int64_t N, int64_t K) {
    return ProductArgs{a, b, amax_a, amax_b, M, N, split_pad(K) / kStepK, tiles_of(M, kTileM), tiles_of(N, kTileN), split_pad(K) / kStepK, 0, Codes{}, nullptr, nullptr};
}
dim3 grid_of_dh(const VocabArgs& v, const LibraryState& lib) { return dim3((unsigned)std::min<int64_t>(tiles_of(v.M * v.D, 1024), 8 * lib.cus)); }
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
    if (tokens == 0) return 0;
    Plan p{};
    FewPlan few{};
    if (few_for_forward(tokens, dim, vocabulary)) few_plan_forward(ws, few, VocabArgs{tokens, vocabulary, dim, nullptr, nullptr, 0, 0, 0.f});
    else plan_forward(ws, p, tokens, dim, vocabulary, true);
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
    Workspace ws(workspace, workspace_bytes);
    if (v.M > 0 && few_for_forward(v.M, v.D, v.V)) {
        FewPlan p{};
        few_plan_forward(ws, p, v);
        if (int rc = ws.check(who)) return rc;
        few_forward(p, v, operand(H), operand(W), stream);
        const JoinArgs jn{v, p.part, label_smoothing > 0.f ? p.part_x : nullptr, p.target_logit, p.tiles, per_sample_loss, lse, v.M <= 64 ? loss_sum : nullptr, valid_count};
        hipLaunchKernelGGL(vocab_join_kernel, dim3((unsigned)tiles_of(v.M, 64)), dim3(1024), 0, stream, jn);
    } else if (v.M > 0) {
        const bool word_rows = rows_of_words(W);
        Plan p{};
        plan_forward(ws, p, v.M, v.D, v.V, word_rows);
        if (int rc = ws.check(who)) return rc;
        launch_split(p, H, W, v, Upstream{}, call.state);
        const ProductArgs g = product(p.w, p.amax_w, p.h, nullptr, v.V, v.M, v.D);
        LogitArgs a{};
        a.v = v; a.words = v.V; a.h_inverse = p.h_inverse; a.part = p.part; a.part_x = label_smoothing > 0.f ? p.part_x : nullptr; a.target_logit = p.target_logit;
        if (word_rows) hipLaunchKernelGGL((vocab_logits_kernel<true, false>), grid_of(g), dim3(256), 0, stream, g, a);
        else hipLaunchKernelGGL((vocab_logits_kernel<false, false>), grid_of(g), dim3(256), 0, stream, g, a);
        const JoinArgs jn{v, p.part, a.part_x, p.target_logit, g.tiles_m, per_sample_loss, lse, v.M <= 64 ? loss_sum : nullptr, valid_count};
        hipLaunchKernelGGL(vocab_join_kernel, dim3((unsigned)tiles_of(v.M, 64)), dim3(1024), 0, stream, jn);
    }
    if (v.M == 0 || v.M > 64) hipLaunchKernelGGL(vocab_total_kernel, dim3(1), dim3(1024), 0, stream, v, per_sample_loss, loss_sum, valid_count);
    return call.finish(sync);
}

int64_t tenmo_hip_vocabulary_loss_backward_workspace_bytes(int64_t tokens, int64_t dim, int64_t vocabulary) {
    if (int rc = check_sizes(tokens, dim, vocabulary, "tenmo_hip_vocabulary_loss_backward_workspace_bytes")) return rc;
    Workspace ws(nullptr, 0);
    if (tokens == 0) return 0;
    Plan p{};
    FewPlan few{};
    if (few_for_backward(tokens, dim, vocabulary)) few_plan_backward(ws, few, VocabArgs{tokens, vocabulary, dim, nullptr, nullptr, 0, 0, 0.f});
    else plan_backward(ws, p, tokens, dim, vocabulary, true);
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
    float* gw = grad_W ? const_cast<float*>(grad_W->data) + grad_W->offset : nullptr;
    const int64_t gw_d = grad_W ? grad_W->strides[0] : 0, gw_v = grad_W ? grad_W->strides[1] : 0;
    const bool word_rows = rows_of_words(W), dw_by_words = gw_d == 1 || gw_v != 1;
    Workspace ws(workspace, workspace_bytes);
    const Upstream up{upstream, (int)reduction, valid_count};
    if (v.M > 0 && few_for_backward(v.M, v.D, v.V)) {
        FewPlan p{};
        few_plan_backward(ws, p, v);
        if (int rc = ws.check(who)) return rc;
        few_backward(p, v, operand(H), operand(W), lse, up, grad_H != nullptr, gw, gw_d, gw_v, grad_bias, add, stream);
        if (grad_H) hipLaunchKernelGGL(vocab_dh_kernel, grid_of_dh(v, call.state), dim3(256), 0, stream, p.part_h, p.runs, v, up, grad_H, add);
        return call.finish(sync);
    }
    auto grid_of_dw = [&](int64_t values) { return dim3((unsigned)std::min<int64_t>(tiles_of(values, 256), 8 * call.state.cus)); };
    if (v.M == 0) { // nothing is added up
        if (grad_W && !add) hipLaunchKernelGGL(vocab_dw_kernel, grid_of_dw(v.V * v.D), dim3(256), 0, stream, nullptr, 0, v.V, v.D, StoreArgs{gw, gw_v, gw_d, 0});
        if (grad_bias) hipLaunchKernelGGL(vocab_db_kernel, dim3((unsigned)tiles_of(v.V, 256)), dim3(256), 0, stream, nullptr, 0, v.V, grad_bias, add);
        return call.finish(sync);
    }
    Plan p{};
    plan_backward(ws, p, v.M, v.D, v.V, word_rows);
    if (int rc = ws.check(who)) return rc;
    launch_split(p, H, W, v, up, call.state);
    int64_t runs = 0;
    for (int64_t first = 0; first < v.V; first += p.piece) {
        const int64_t words = std::min(p.piece, v.V - first);
        SplitMatrix G = p.g, GW = p.gw;
        G.pitch = GW.pitch = split_pad(words);
        const SplitMatrix w = words_of(p.w, first, word_rows);
        const ProductArgs g = product(w, p.amax_w, p.h, nullptr, words, v.M, v.D);
        LogitArgs a{};
        a.v = v; a.first = first; a.words = words; a.h_inverse = p.h_inverse; a.lse = lse; a.up = up; a.part_db = grad_bias ? p.part_db : nullptr;
        if (grad_H) a.g = G;
        if (grad_W) a.gw = GW, a.word_class = p.word_class, a.top_f = p.top_f;
        if (word_rows) hipLaunchKernelGGL((vocab_logits_kernel<true, true>), grid_of(g), dim3(256), 0, stream, g, a);
        else hipLaunchKernelGGL((vocab_logits_kernel<false, true>), grid_of(g), dim3(256), 0, stream, g, a);
        if (grad_W)
            hipLaunchKernelGGL(vocab_unit_kernel, dim3((unsigned)tiles_of(GW.pitch, 256)), dim3(256), 0, stream, p.word_class, GW.pitch, tiles_of(v.M, kCodeK), p.codes, p.unit);
        ProductArgs dh{}, dw{};
        StoreArgs sh{}, sw{};
        int64_t h_tiles = 0, w_tiles = 0;
        if (grad_H) {
            dh = product(G, nullptr, words_of(p.w, first, word_rows), p.amax_w, v.M, v.D, words);
            dh.run_steps = tiles_of(tiles_of(p.piece, kStepK), p.runs); // (of the whole piece: a last one that is shorter has as many or fewer runs)
            dh.run_stride = v.M * v.D;
            sh = StoreArgs{p.part_h, v.D, 1, first > 0};
            h_tiles = dh.tiles_m * dh.tiles_n * tiles_of(dh.k_steps, dh.run_steps);
            runs = std::max(runs, tiles_of(dh.k_steps, dh.run_steps));
        }
        if (grad_W) { // as [words][D] or [D][words], whichever puts the axis with unit stride across the lanes
            float* to = gw + first * gw_v;
            if (dw_by_words) {
                dw = product(GW, nullptr, p.h, nullptr, words, v.D, v.M);
                sw = StoreArgs{to, gw_v, gw_d, add};
            } else {
                dw = product(p.h, nullptr, GW, nullptr, v.D, words, v.M);
                sw = StoreArgs{to, gw_d, gw_v, add};
            }
            dw.codes = Codes{p.codes, GW.pitch};
            dw.unit = p.unit;
            dw.top_f = p.top_f;
            w_tiles = dw.tiles_m * dw.tiles_n;
        }
        const StoreArgs to_w = sw;
        int64_t w_runs = 1;
        if (grad_W && p.w_runs > 1) {
            dw.run_steps = tiles_of(dw.k_steps, p.w_runs);
            dw.run_stride = dw.M * dw.N;
            w_runs = tiles_of(dw.k_steps, dw.run_steps);
            w_tiles *= w_runs;
            sw = StoreArgs{p.part_w, dw.N, 1, 0};
        }
        if (h_tiles + w_tiles == 0) continue;
        const dim3 grid((unsigned)(h_tiles + w_tiles));
        if (word_rows && dw_by_words) hipLaunchKernelGGL((vocab_products_kernel<false, true>), grid, dim3(256), 0, stream, dh, sh, (uint32_t)h_tiles, dw, sw);
        else if (word_rows) hipLaunchKernelGGL((vocab_products_kernel<false, false>), grid, dim3(256), 0, stream, dh, sh, (uint32_t)h_tiles, dw, sw);
        else if (dw_by_words) hipLaunchKernelGGL((vocab_products_kernel<true, true>), grid, dim3(256), 0, stream, dh, sh, (uint32_t)h_tiles, dw, sw);
        else hipLaunchKernelGGL((vocab_products_kernel<true, false>), grid, dim3(256), 0, stream, dh, sh, (uint32_t)h_tiles, dw, sw);
        if (grad_W && p.w_runs > 1)
            hipLaunchKernelGGL(vocab_dw_kernel, grid_of_dw(dw.run_stride), dim3(256), 0, stream, p.part_w, w_runs, dw.M, dw.N, to_w);
    }
    if (grad_H)
        hipLaunchKernelGGL(vocab_dh_kernel, grid_of_dh(v, call.state), dim3(256), 0, stream, p.part_h, runs, v, up, grad_H, add);
    if (grad_bias) hipLaunchKernelGGL(vocab_db_kernel, dim3((unsigned)tiles_of(v.V, 256)), dim3(256), 0, stream, p.part_db, 2 * tiles_of(v.M, kTileN), v.V, grad_bias, add);
    return call.finish(sync);
}

} // extern "C"
