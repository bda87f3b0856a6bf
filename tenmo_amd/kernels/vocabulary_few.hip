// The vocabulary loss for few tokens, or a small W: what bounds it is reading W (and writing dW), or latency, so W is read as it is, in fp32, by the fp32 matrix instruction.
//
//   forward   x = H W: a workgroup for 128 words and 32 tokens, or 64 and 64, over all of D; its maximum and sum of each token leave the chip.
//   backward  the same product again, ending as G in fp32 [tokens, words]; dH = G W^T, the words cut into runs with a sum each;
//             dW = (scale H)^T G, tiles of 128 x 64, the tokens in blocks of 64 through LDS.
//
// The split form of the products (vocabulary.hip) reads W three times and writes it once before it begins, which its rate pays back only for many tokens and a large W.  Forward and
// backward with W as an embedding [words, D], here against the split form:
//       768 x 50257:    1 token 52 + 126 us against 146 + 271;   64 tokens 74 + 190 against 142 + 266;   256 tokens 221 + 610 against 173 + 367
//      1600 x 4000:    64 tokens 50 +  87 us against  91 + 128;  256 tokens 53 + 146 against  91 + 167;  512 tokens  85 + 248 against  92 + 188
//       128 x 1000:    64 tokens 19 +  22 us against  31 +  45;  256 tokens 25 +  41 against  30 +  52;  512 tokens  25 +  61 against  30 +  54
// One read of the first W (154 MB) takes 30 us at the rate of a copy, its backward (W twice, dW once) 92 us.
// Both products with W have the matrix in the rows of the instruction's result and the tokens in its columns: rows r of 32 in LDS, K-major ([row][k], 32 k and 4 of padding: a
// float4 of four k a lane, 16 rows in 16 different bank groups) where the memory runs along k, MN-major ([k][row]) where it runs along r.
#include "vocabulary.hpp"

#include <algorithm>

namespace tenmo {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int KC = 32;       // k a step
constexpr int PITCH = KC + 4;

enum { kLoss, kGrad, kHidden };

struct FewArgs {
    VocabArgs v;
    Operand2 a;          // rows x k: W transposed, or W
    int64_t rows, k;     // rows of the result: words, or D
    Operand2 b;          // tokens x k: H, or G
    int64_t run;         // k of a run
    float2* part;
    float *part_x, *target_logit;
    const float* lse;
    float* out;          // G [tokens][words], or [runs][tokens][D]
};

// ROWS x KC of an operand on the way into LDS, ROWS * KC / 256 values a thread
template <int ROWS, bool KMAJOR>
struct Staged {
    static constexpr int N = ROWS * KC / 1024; // groups of four
    f32x4 x[N];
    // Rows behind the last are the last again (their products are not stored).  No branch of a lane's own: one would wait for the loads before it.
    __device__ __forceinline__ void load(const Operand2& o, int64_t r0, int64_t rows, int64_t k0, int64_t k_end) {
        const bool wide = KMAJOR ? o.c == 1 && k0 + KC <= k_end : o.r == 1 && r0 + ROWS <= rows;
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int y = threadIdx.x + 256 * i;
                const int64_t r = r0 + (KMAJOR ? y / (KC / 4) : y % (ROWS / 4) * 4), k = k0 + (KMAJOR ? y % (KC / 4) * 4 : y / (ROWS / 4));
                x[i] = *(const f32x4_u*)(o.p + (KMAJOR && r >= rows ? rows - 1 : r) * o.r + (!KMAJOR && k >= k_end ? k_end - 1 : k) * o.c);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int y = threadIdx.x + 256 * i;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t r = r0 + (KMAJOR ? y / (KC / 4) : y % (ROWS / 4) * 4 + e), k = k0 + (KMAJOR ? y % (KC / 4) * 4 + e : y / (ROWS / 4));
                    x[i][e] = o.p[(r >= rows ? rows - 1 : r) * o.r + (k >= k_end ? k_end - 1 : k) * o.c];
                }
            }
        }
    }
    // k of what was loaded, and its end: zeros behind it
    __device__ __forceinline__ void store(float* lds, int64_t k0, int64_t k_end) {
        if (k0 + KC > k_end)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int y = threadIdx.x + 256 * i;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = k0 + (KMAJOR ? y % (KC / 4) * 4 + e : y / (ROWS / 4)) < k_end ? x[i][e] : 0.f;
            }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int y = threadIdx.x + 256 * i;
            if (KMAJOR) *(f32x4*)(lds + y / (KC / 4) * PITCH + y % (KC / 4) * 4) = x[i];
            else *(f32x4*)(lds + y / (ROWS / 4) * (ROWS + 4) + y % (ROWS / 4) * 4) = x[i];
        }
    }
    static constexpr int FLOATS = KMAJOR ? ROWS * PITCH : KC * (ROWS + 4);
    // the four k of this half of the wavefront, of eight from k8, for row `row`
    static __device__ __forceinline__ f32x4 read(const float* lds, int row, int k8, int half) {
        if (KMAJOR) return *(const f32x4*)(lds + row * PITCH + k8 + 4 * half);
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = lds[(k8 + 4 * half + e) * (ROWS + 4) + row];
        return y;
    }
};

template <int TOKENS, bool A_KMAJOR>
struct FewTile {
    static constexpr int ROWS = TOKENS == 32 ? 128 : 64;
    using A = Staged<ROWS, A_KMAJOR>;
    using B = Staged<TOKENS, true>;
    static constexpr int FLOATS = 2 * (A::FLOATS + B::FLOATS);
};

template <int TOKENS, int MODE, bool A_KMAJOR>
__device__ __forceinline__ void few_product(const FewArgs& a, int64_t group, float* lds) {
    using Tile = FewTile<TOKENS, A_KMAJOR>;
    constexpr int ROWS = Tile::ROWS;
    using A = typename Tile::A;
    using B = typename Tile::B;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int row_block = TOKENS == 32 ? wave : wave & 1, token_block = TOKENS == 32 ? 0 : wave >> 1;
    // the blocks of tokens that share a tile of W lie next to each other
    const int64_t tiles = (a.rows + ROWS - 1) / ROWS, token_blocks = (a.v.M + TOKENS - 1) / TOKENS, id = group / token_blocks;
    const int64_t t0 = (group - id * token_blocks) * TOKENS, run = MODE == kHidden ? id / tiles : 0, tile = id - run * tiles;
    const int64_t r0 = tile * ROWS, k0 = run * a.run, k_end = MODE == kHidden && k0 + a.run < a.k ? k0 + a.run : a.k;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    A sa;
    B sb;
    sa.load(a.a, r0, a.rows, k0, k_end);
    sb.load(a.b, t0, a.v.M, k0, k_end);
    int stage = 0;
    for (int64_t k = k0; k < k_end; k += KC, stage ^= 1) {
        float *const lds_a = lds + stage * A::FLOATS, *const lds_b = lds + 2 * A::FLOATS + stage * B::FLOATS;
        sa.store(lds_a, k, k_end);
        sb.store(lds_b, k, k_end);
        __syncthreads();
        if (k + KC < k_end) { // on the way while this step is multiplied; its place in LDS was read a step ago
            sa.load(a.a, r0, a.rows, k + KC, k_end);
            sb.load(a.b, t0, a.v.M, k + KC, k_end);
        }
#pragma unroll
        for (int k8 = 0; k8 < KC; k8 += 8) {
            const f32x4 x = A::read(lds_a, 32 * row_block + (lane & 31), k8, half), y = B::read(lds_b, 32 * token_block + (lane & 31), k8, half);
#pragma unroll
            for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[s], y[s], acc, 0, 0, 0);
        }
    }
    // register e: row 8 (e / 4) + 4 half + e % 4 of the block, column lane % 32
    const int64_t row0 = r0 + 32 * row_block + 4 * half, token = t0 + 32 * token_block + (lane & 31);
    if (MODE == kHidden) {
        if (token >= a.v.M) return;
        float* to = a.out + (run * a.v.M + token) * a.rows;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t r = row0 + 8 * q;
            if (r + 3 < a.rows) *(f32x4_u*)(to + r) = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r + e < a.rows) to[r + e] = acc[4 * q + e];
        }
        return;
    }
    const int64_t at = (token < a.v.M ? target_of(a.v, token) : a.v.ignore) - row0; // the target's place from this lane's first word
    if (a.v.bias)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t r = row0 + 8 * (e >> 2) + (e & 3);
            if (r < a.rows) acc[e] += a.v.bias[r];
        }
    if (MODE == kLoss) {
        __shared__ float join[3][ROWS / 32][TOKENS];
        float top = -__builtin_inff(), sum = 0.f, sx = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const bool in = row0 + 8 * (e >> 2) + (e & 3) < a.rows;
            sx += in ? acc[e] : 0.f;
            acc[e] = in ? acc[e] : -__builtin_inff();
            top = fmaxf(top, acc[e]);
        }
        top = halves_max(top);
        const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sum += __expf(acc[e] - base);
            if (token < a.v.M && at == 8 * (e >> 2) + (e & 3)) a.target_logit[token] = acc[e];
        }
        sum = halves_sum(sum);
        sx = halves_sum(sx);
        const int col = 32 * token_block + (lane & 31);
        if (half == 0) join[0][row_block][col] = top, join[1][row_block][col] = sum, join[2][row_block][col] = sx;
        __syncthreads();
        const int t = threadIdx.x;
        if (t < TOKENS && t0 + t < a.v.M) {
            float m = join[0][0][t], s = 0.f, x = 0.f;
#pragma unroll
            for (int w = 1; w < ROWS / 32; ++w) m = fmaxf(m, join[0][w][t]);
            const float b = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
            for (int w = 0; w < ROWS / 32; ++w) s += join[1][w][t] * __expf(join[0][w][t] - b), x += join[2][w][t];
            a.part[tile * a.v.M + t0 + t] = make_float2(m, s);
            if (a.part_x) a.part_x[tile * a.v.M + t0 + t] = x;
        }
        return;
    }
    if (token >= a.v.M) return;
    const bool valid = target_of(a.v, token) != a.v.ignore;
    const float lse = a.lse[token], smooth = a.v.ls / (float)a.v.V;
    float* to = a.out + token * a.v.V;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        f32x4 g;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            g[e] = __expf(acc[4 * q + e] - lse) - smooth;
            if (at == 8 * q + e) g[e] -= 1.f - a.v.ls;
            g[e] = valid ? g[e] : 0.f;
        }
        const int64_t r = row0 + 8 * q;
        if (r + 3 < a.rows) *(f32x4_u*)(to + r) = g;
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r + e < a.rows) to[r + e] = g[e];
    }
}

template <int TOKENS, int MODE, bool A_KMAJOR>
__global__ __launch_bounds__(256) void few_kernel(const FewArgs a) {
    __shared__ __align__(16) float lds[FewTile<TOKENS, A_KMAJOR>::FLOATS];
    few_product<TOKENS, MODE, A_KMAJOR>(a, blockIdx.x, lds);
}

// dW: rows i of the result (words, or D) by columns j, the one with unit stride; X [tokens][i] and Y [tokens][j] in LDS whole
struct FewWeight {
    VocabArgs v;
    Upstream up;
    Operand2 x, y;
    int x_is_h;       // the hidden states are X, or else Y: their rows are multiplied by their factors
    int64_t rows, cols;
    float* out;
    int64_t rs, cs;
    int accumulate;
};

// columns c0 .. c0 + WIDTH of every token, on the way into LDS
template <int TOKENS, int WIDTH>
struct TokenRows {
    static constexpr int N = TOKENS * WIDTH / 1024;
    f32x4 x[N];
    // tokens t0 ..; columns behind the last are the last again (their products are not stored), and so are tokens
    __device__ __forceinline__ void load(const Operand2& o, int64_t t0, int64_t tokens, int64_t c0, int64_t cols) {
        const bool wide = o.c == 1 && c0 + WIDTH <= cols;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int y = threadIdx.x + 256 * i, m = y / (WIDTH / 4);
            const int64_t c = c0 + y % (WIDTH / 4) * 4;
            const float* p = o.p + (t0 + m >= tokens ? tokens - 1 : t0 + m) * o.r;
            if (wide) x[i] = *(const f32x4_u*)(p + c);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = p[(c + e >= cols ? cols - 1 : c + e) * o.c];
        }
    }
    // times the rows' factors: rows without a part in the gradient are zeros, whatever they hold
    __device__ __forceinline__ void store(float* lds, const float* factors) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int y = threadIdx.x + 256 * i, m = y / (WIDTH / 4);
            const float f = factors[m];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = f == 0.f ? 0.f : x[i][e] * f;
            *(f32x4*)(lds + m * (WIDTH + 4) + y % (WIDTH / 4) * 4) = x[i];
        }
    }
};

constexpr int kWeightI = 128, kWeightJ = 64;
template <int TOKENS>
constexpr int kWeightFloats = TOKENS * (kWeightI + 4 + kWeightJ + 4 + 2);

template <int TOKENS>
__device__ __forceinline__ void few_weight(const FewWeight& a, int64_t id, float* lds) {
    constexpr int I = kWeightI, J = kWeightJ;
    float *const lx = lds, *const ly = lds + TOKENS * (I + 4), *const factors = ly + TOKENS * (J + 4); // [0 ..] of G: one for every token; [TOKENS ..] of H
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int64_t tiles_j = (a.cols + J - 1) / J, i0 = id / tiles_j * I, j0 = id % tiles_j * J;
    TokenRows<TOKENS, I> x;
    TokenRows<TOKENS, J> y;
    f32x16 acc[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] = 0.f;
    x.load(a.x, 0, a.v.M, i0, a.rows);
    y.load(a.y, 0, a.v.M, j0, a.cols);
    for (int64_t t0 = 0; t0 < a.v.M; t0 += TOKENS) {
        if (threadIdx.x < TOKENS) { // each once: it hangs on three loads in a row
            const int64_t m = t0 + threadIdx.x;
            factors[threadIdx.x] = m < a.v.M ? 1.f : 0.f;
            factors[TOKENS + threadIdx.x] = m < a.v.M ? row_factor(a.v, a.up, m) : 0.f;
        }
        __syncthreads(); // (and the block before is multiplied)
        x.store(lx, factors + (a.x_is_h ? TOKENS : 0));
        y.store(ly, factors + (a.x_is_h ? 0 : TOKENS));
        __syncthreads();
        if (t0 + TOKENS < a.v.M) {
            x.load(a.x, t0 + TOKENS, a.v.M, i0, a.rows);
            y.load(a.y, t0 + TOKENS, a.v.M, j0, a.cols);
        }
#pragma unroll 4
        for (int m = 0; m < TOKENS; m += 2) {
            const float left = lx[(m + half) * (I + 4) + 32 * wave + (lane & 31)];
#pragma unroll
            for (int b = 0; b < 2; ++b) acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(left, ly[(m + half) * (J + 4) + 32 * b + (lane & 31)], acc[b], 0, 0, 0);
        }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t i = i0 + 32 * wave + 8 * (e >> 2) + 4 * half + (e & 3), j = j0 + 32 * b + (lane & 31);
            if (i >= a.rows || j >= a.cols) continue;
            float* to = a.out + i * a.rs + j * a.cs;
            *to = a.accumulate ? *to + acc[b][e] : acc[b][e];
        }
}

// dH's runs (the first workgroups) and dW in one launch: neither needs the other
template <int TOKENS, bool A_KMAJOR>
__global__ __launch_bounds__(256) void few_gradients_kernel(const FewArgs h, uint32_t h_groups, const FewWeight w) {
    constexpr int FLOATS = FewTile<TOKENS, A_KMAJOR>::FLOATS > kWeightFloats<TOKENS> ? FewTile<TOKENS, A_KMAJOR>::FLOATS : kWeightFloats<TOKENS>;
    __shared__ __align__(16) float lds[FLOATS];
    if (blockIdx.x < h_groups) few_product<TOKENS, kHidden, A_KMAJOR>(h, blockIdx.x, lds);
    else few_weight<TOKENS>(w, blockIdx.x - h_groups, lds);
}

// db of 64 words: each of the 16 wavefronts takes every 16th token, then their sums are added in order
__global__ __launch_bounds__(1024) void few_bias_kernel(const VocabArgs v, const Upstream up, const float* __restrict g, float* db, int accumulate) {
    __shared__ float sums[16][64], factors[1024];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t word = (int64_t)blockIdx.x * 64 + lane, column = word < v.V ? word : v.V - 1;
    float s = 0.f;
    for (int64_t m0 = 0; m0 < v.M; m0 += 1024) {
        if (m0) __syncthreads();
        if (m0 + threadIdx.x < v.M) factors[threadIdx.x] = row_factor(v, up, m0 + threadIdx.x);
        __syncthreads();
        const int many = v.M - m0 < 1024 ? (int)(v.M - m0) : 1024;
#pragma unroll 8
        for (int m = wave; m < many; m += 16) s += g[(m0 + m) * v.V + column] * factors[m];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave || word >= v.V) return;
    for (int w = 1; w < 16; ++w) s += sums[w][lane];
    db[word] = accumulate ? db[word] + s : s;
}

int64_t up_to(int64_t n, int64_t t) { return (n + t - 1) / t; }
// Four wavefronts of 32 x 32 each: four of words and one of tokens, or two and two.  That is a workgroup for every 128 words of up to 32 tokens, each with the whole of D as its chain: fewer than there are
// CUs where the words are few (1600 x 8000: 63 of them, 64 us forward for 1 to 32 tokens, 47 for 33 to 64 by 125 workgroups); 768 x 50257: 52 and 74 us.
int64_t rows_a_tile(int64_t tokens) { return tokens <= 32 ? 128 : 64; }

int64_t token_blocks(int64_t tokens) { return tokens <= 32 ? 1 : up_to(tokens, 64); }

bool k_major(const FewArgs& a) { return a.a.c == 1 || a.a.r != 1; }

template <int MODE>
void launch_few(const FewArgs& a, int64_t tiles, hipStream_t stream) {
    const int64_t grid = tiles * token_blocks(a.v.M);
    if (a.v.M <= 32) {
        if (k_major(a)) hipLaunchKernelGGL((few_kernel<32, MODE, true>), dim3((unsigned)grid), dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((few_kernel<32, MODE, false>), dim3((unsigned)grid), dim3(256), 0, stream, a);
    } else {
        if (k_major(a)) hipLaunchKernelGGL((few_kernel<64, MODE, true>), dim3((unsigned)grid), dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((few_kernel<64, MODE, false>), dim3((unsigned)grid), dim3(256), 0, stream, a);
    }
}

} // namespace

// By the values of W that blocks of 64 tokens read, fitted to 237 sizes (64 to 16384 tokens, 32 to 1600 dimensions, 300 to 50257 words): no choice costs more than 1.09 of the other;
// backward each block of tokens also takes a turn in dW's sum.
bool few_for_forward(int64_t tokens, int64_t dim, int64_t words) {
    return tokens <= 64 || (double)token_blocks(tokens) * dim * words <= 8e6 + 20e3 * dim + 1.6 * dim * words;
}
bool few_for_backward(int64_t tokens, int64_t dim, int64_t words) {
    return tokens <= 64 || token_blocks(tokens) * ((double)dim * words + 3e6) <= 20e6 + 20e3 * dim + 0.5 * dim * words;
}

void few_plan_forward(Workspace& ws, FewPlan& p, const VocabArgs& v) {
    p.tiles = up_to(v.V, rows_a_tile(v.M));
    p.part = ws.take<float2>(p.tiles * v.M);
    p.part_x = ws.take<float>(p.tiles * v.M);
    p.target_logit = ws.take<float>(v.M);
}

void few_plan_backward(Workspace& ws, FewPlan& p, const VocabArgs& v) {
    p.g = ws.take<float>(v.M * v.V);
    // two workgroups a CU, of at least 64 words each
    p.run = up_to(up_to(v.V, std::max<int64_t>(1, std::min(512 / (up_to(v.D, rows_a_tile(v.M)) * token_blocks(v.M)), v.V / 64))), KC) * KC;
    p.runs = up_to(v.V, p.run);
    p.part_h = ws.take<float>(p.runs * v.M * v.D);
}

void few_forward(const FewPlan& p, const VocabArgs& v, const Operand2& h, const Operand2& w, hipStream_t stream) {
    FewArgs a{};
    a.v = v;
    a.a = Operand2{w.p, w.c, w.r}; a.rows = v.V; a.k = v.D; a.b = h;
    a.part = p.part; a.part_x = v.ls > 0.f ? p.part_x : nullptr; a.target_logit = p.target_logit;
    launch_few<kLoss>(a, p.tiles, stream);
}

void few_backward(const FewPlan& p, const VocabArgs& v, const Operand2& h, const Operand2& w, const float* lse, const Upstream& up, bool want_h,
                  float* grad_w, int64_t gw_d, int64_t gw_v, float* grad_bias, int accumulate, hipStream_t stream) {
    FewArgs a{};
    a.v = v; a.lse = lse;
    a.a = Operand2{w.p, w.c, w.r}; a.rows = v.V; a.k = v.D; a.b = h;
    a.out = p.g;
    launch_few<kGrad>(a, up_to(v.V, rows_a_tile(v.M)), stream);
    const Operand2 g{p.g, v.V, 1};
    a.a = w; a.rows = v.D; a.k = v.V; a.b = g;
    a.run = p.run;
    a.out = p.part_h;
    FewWeight f{};
    f.v = v; f.up = up; f.out = grad_w; f.accumulate = accumulate;
    if (gw_d == 1 || gw_v != 1) { f.x = g; f.y = h; f.rows = v.V; f.cols = v.D; f.rs = gw_v; f.cs = gw_d; }
    else { f.x = h; f.y = g; f.x_is_h = 1; f.rows = v.D; f.cols = v.V; f.rs = gw_d; f.cs = gw_v; }
    const int64_t h_groups = want_h ? up_to(v.D, rows_a_tile(v.M)) * p.runs * token_blocks(v.M) : 0, w_groups = grad_w ? up_to(f.rows, kWeightI) * up_to(f.cols, kWeightJ) : 0;
    if (h_groups + w_groups > 0) {
        const dim3 grid((unsigned)(h_groups + w_groups));
        if (v.M <= 32) {
            if (k_major(a)) hipLaunchKernelGGL((few_gradients_kernel<32, true>), grid, dim3(256), 0, stream, a, (uint32_t)h_groups, f);
            else hipLaunchKernelGGL((few_gradients_kernel<32, false>), grid, dim3(256), 0, stream, a, (uint32_t)h_groups, f);
        } else {
            if (k_major(a)) hipLaunchKernelGGL((few_gradients_kernel<64, true>), grid, dim3(256), 0, stream, a, (uint32_t)h_groups, f);
            else hipLaunchKernelGGL((few_gradients_kernel<64, false>), grid, dim3(256), 0, stream, a, (uint32_t)h_groups, f);
        }
    }
    if (grad_bias) hipLaunchKernelGGL(few_bias_kernel, dim3((unsigned)up_to(v.V, 64)), dim3(1024), 0, stream, v, up, p.g, grad_bias, accumulate);
}

} // namespace tenmo
