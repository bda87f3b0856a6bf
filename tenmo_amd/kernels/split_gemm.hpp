// fp32 products on the fp16 matrix units: operands as two halves.
//
// The fp32 matrix instruction of gfx950 does 64 multiply-adds a cycle and SIMD, the fp16 one 512.  A value scaled by a power of two (so that the
// largest of its matrix lies in [2^14, 2^15)) is held as h + l with h = fp16(x), l = fp16(x - h); then a b = h_a h_b + h_a l_b + l_a h_b up to
//   |x - h - l| <= 2^-22 |x| (or 2^-25 where l is subnormal: 2^-40 of the matrix's largest value, the matrix units keep subnormals) and
//   |l_a l_b| <= 2^-22 |a b|,
// the size of the roundings of an fp32 accumulation (the matrix units add in fp32): three fp16 products give an fp32 product at 512 / 3 = 2.7 times the
// fp32 instruction's rate.  This is the error-corrected half-precision product of Ootomo and Yokota (2022).
// Values that are not finite have l = 0 and make every sum they enter not finite.
//
// Split matrix: rows of `pitch` values (a multiple of 16), each 8 of them 32 bytes: 8 h, then 8 l; as many bytes as the fp32 matrix.
// Rows are padded to a multiple of 16 and both paddings hold zeros.
#ifndef TENMO_KERNELS_SPLIT_GEMM_HPP
#define TENMO_KERNELS_SPLIT_GEMM_HPP
#include "../csrc/gfx950_asm.hpp"
#include "entry.hpp"

namespace tenmo {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct SplitMatrix {
    float* p;       // 16 bytes = 8 halves of one kind
    int64_t pitch;  // values a row
    int64_t rows;   // without padding
};

__host__ __device__ inline int64_t split_pad(int64_t n) { return (n + 15) / 16 * 16; }

// ---- scale and split --------------------------------------------------------------------------------------------------------

constexpr int kAmaxParts = 512; // partial maxima of one matrix

// the largest finite magnitude among the bit patterns
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
    const uint32_t m = __float_as_uint(x) & 0x7fffffffu;
    return m < 0x7f800000u ? m : 0u;
}
// (of magnitudes: their order as floats is that of their bits)
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) { return __float_as_uint(wave_max(__uint_as_float(v))); }
// The power of two that brings the magnitude with these bits into [2^14, 2^15); 1 for zero.
__device__ __forceinline__ float split_scale(uint32_t bits) {
    if (bits == 0) return 1.f;
    int e = (int)(bits >> 23) - 127; // subnormals: -127, their values end up smaller
    e = 14 - e;
    return __uint_as_float((uint32_t)((e > 126 ? 126 : e) + 127) << 23); // e >= 14 - 127
}

// (x is the last operation's fp32 result in both uses, or exact: the compiler may otherwise round a product to fp16 by two ways)
__device__ __forceinline__ void split_value(float x, _Float16& h, _Float16& l) {
    asm("" : "+v"(x));
    h = (_Float16)x;
    const float r = x - (float)h;
    l = (_Float16)(r - r == 0.f ? r : 0.f); // x not finite: h alone
}
// a 1 that the compiler takes for a variable: x * one - h, rounded to fp16, is one mixed-precision instruction, x - h converts twice
__device__ __forceinline__ float variable_one() {
    float one = 1.f;
    asm volatile("" : "+v"(one));
    return one;
}
// ---- the product ----------------------------------------------------------------------------------------------------------------

// C[m, n] = sum over k of A[m, k] B[k, n] for a tile of 256 x 128 and the K steps k_first .., wavefronts 2 x 2, K in steps of 16 through a ring of three stages in LDS
// (24 KiB each: two workgroups a CU), filled by direct global -> LDS loads two steps ahead, one barrier a step.
// An operand is K-major (row m, or n, of the split matrix holds its K values) or MN-major (row k holds the values of all m, or n):
//   * K-major stage: [row][4 chunks of 16 bytes], chunk c = 2 * (k / 8) + kind (0: h, 1: l) at slot c ^ ((row / 4) & 3): the 16 rows that a quarter of a
//     wavefront reads lie in 16 different slots of the 256 bytes of banks.
//   * MN-major stage: [k][columns / 4 chunks], chunk c = 2 * (column / 8) + kind at slot c ^ (k & 1 | (k & 2) << 2), fetched with the transposing LDS
//     read (a group of 16 lanes reads 4 rows of 16 values, each lane receives one column's 4): 4 rows x 4 chunks in 16 different slots.
// Rows and columns beyond the matrix repeat the last one (their results are not stored); K is padded with zeros by the split.
constexpr int kTileM = 256, kTileN = 128, kStepK = 16;
constexpr int kStageBytes = (kTileM + kTileN) * kStepK * 4;
constexpr int kStages = 3;

// an operand's tile as the loads see it
template <int ROWS, bool KMAJOR>
struct TileLoader {
    static constexpr int BLOCKS = ROWS * 64 / 1024 / 4; // 1 KiB loads a wavefront and stage
    uint32_t lane_off[BLOCKS];
    const float* base;
    int64_t step; // floats from one K step to the next

    __device__ __forceinline__ void init(const SplitMatrix& m, int64_t first, int64_t count, int wave, int lane) { // rows (K-major) or columns first .. of `count`
        if (KMAJOR) {
            base = m.p + first * m.pitch;
            step = kStepK;
        } else {
            base = m.p + first;
            step = kStepK * m.pitch;
        }
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i) {
            const int block = wave * BLOCKS + i;
            if (KMAJOR) {
                const int row = block * 16 + lane / 4, chunk = (lane & 3) ^ ((row >> 2) & 3);
                const int64_t r = first + row < count ? row : count - 1 - first;
                lane_off[i] = (uint32_t)(r * m.pitch * 4 + chunk * 16);
            } else {
                constexpr int CHUNKS = ROWS / 4; // a row
                const int k = block * 64 / CHUNKS + lane / CHUNKS, chunk = (lane % CHUNKS) ^ ((k & 1) | (k & 2) << 2);
                const int64_t pad = split_pad(count) - first; // columns that exist, zeros among them
                const int64_t c = (chunk / 2) * 8 < pad ? chunk : 2 * (pad / 8 - 1) + (chunk & 1);
                lane_off[i] = (uint32_t)(k * m.pitch * 4 + c * 16);
            }
        }
    }
    __device__ __forceinline__ void load(float* lds, uint32_t at, int wave, int64_t k_step) const {
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i) direct_load_16B(lds, at + (uint32_t)(wave * BLOCKS + i) * 1024u, lane_off[i], base + k_step * step);
    }
};

// a wavefront's fragments of an operand: 32 rows (or columns) x 16 k each
template <int ROWS, bool KMAJOR>
struct TileReader {
    uint32_t off[KMAJOR ? 2 : 4]; // K-major: by kind; MN-major: by kind and parity of the block of 32

    __device__ __forceinline__ void init(uint32_t at, int first, int lane) { // first: the wavefront's first row, a multiple of 64
        if (KMAJOR) {
            const int row = first + (lane & 31), half = lane >> 5;
            for (int kind = 0; kind < 2; ++kind) off[kind] = at + row * 64 + ((2 * half + kind) ^ ((row >> 2) & 3)) * 16;
        } else {
            const int p = lane & 15, sub = (lane >> 4) & 1, half = lane >> 5, kq = p >> 2; // k = 8 half + 4 t + kq
            const int f1 = kq & 1, f8 = (kq & 2) << 2;
            for (int kind = 0; kind < 2; ++kind)
                for (int odd = 0; odd < 2; ++odd)
                    off[2 * kind + odd] = at + (8 * half + kq) * (ROWS * 4) + first * 4 + (((8 * odd) ^ f8) + 4 * sub + 2 * ((p & 3) >> 1) + (kind ^ f1)) * 16 + 8 * (p & 1);
        }
    }
    __device__ __forceinline__ f16x8 read(const char* lds, int block, int kind) const { // block of 32 rows
        if (KMAJOR) return *(const f16x8*)(lds + off[kind] + block * 2048);
        const char* q = lds + off[2 * kind + (block & 1)] + (block >> 1) * 256;
        typedef __attribute__((address_space(3))) i16x4* lds_p;
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)q), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(q + 4 * ROWS * 4));
        union { i16x4 s[2]; f16x8 v; } u;
        u.s[0] = a;
        u.s[1] = b;
        return u.v;
    }
};

// waits until at most N of this wavefront's direct loads are in flight and its LDS reads are done, then for the workgroup
template <int N>
__device__ __forceinline__ void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// An operand whose rows (of the product's M or N) have scales of their own, and others in every kCodeK of K: a row is worked on at the smallest of its scales, of which the others are multiples
// by powers of 2^6, and what is held at those is brought down as it is read.  Four bits for each kCodeK of K, eight of them a word: the power of 2^-6.
// With the largest at 2^8 .. 2^14, what lies below it by more than 2^-33 is lost (l, by itself, from 2^-30 on).  Powers of 2^12 in two bits, and nothing left from the third on, take
// as long (2010 us for both products of half of 8192 x 50257, D = 768), but lose values from 2^-24 of the largest on: 1.5e-4 of a sum over 4100 tokens, one of which is the largest.
constexpr int kCodeK = 64, kCodeBits = 6, kCodesAWord = 8, kMostCode = 7; // (7: h ends below 2^-28, as nothing)
enum { kPlain, kCodedA, kCodedB };
struct Codes {
    const uint32_t* p; // [K / (kCodeK * kCodesAWord)][pitch]
    int64_t pitch;
};
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
struct CodeFactor { // fp16 ends at 2^-24: h takes two factors, l is nothing where the second counts
    f16x2 near, far, low;
    __device__ __forceinline__ void set(uint32_t codes, uint32_t at) {
        const int code = (int)((codes >> (4 * at)) & 15u);
        const _Float16 n = (_Float16)__builtin_amdgcn_ldexpf(1.f, -kCodeBits * (code < 4 ? code : 4)), f = (_Float16)__builtin_amdgcn_ldexpf(1.f, -kCodeBits * (code > 4 ? code - 4 : 0));
        near = f16x2{n, n};
        far = f16x2{f, f};
        low = code > 4 ? f16x2{0, 0} : near;
    }
};
__device__ __forceinline__ f16x8 times(f16x8 x, f16x2 f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f[e & 1];
    return x;
}

template <bool A_KMAJOR, bool B_KMAJOR, int CODED = kPlain>
__device__ __forceinline__ void split_tile(f32x16 (&acc)[4][2], float* lds, const SplitMatrix& A, int64_t m0, int64_t M, const SplitMatrix& B, int64_t n0, int64_t N, int64_t k_first, int64_t k_steps,
                                           const Codes& codes = Codes{}) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TileLoader<kTileM, A_KMAJOR> la;
    TileLoader<kTileN, B_KMAJOR> lb;
    la.init(A, m0, M, wave, lane);
    lb.init(B, n0, N, wave, lane);
    TileReader<kTileM, A_KMAJOR> ra;
    TileReader<kTileN, B_KMAJOR> rb;
    ra.init(0, (wave & 1) * 128, lane);
    rb.init(kTileM * kStepK * 4, (wave >> 1) * 64, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    constexpr int LOADS = TileLoader<kTileM, A_KMAJOR>::BLOCKS + TileLoader<kTileN, B_KMAJOR>::BLOCKS;
    auto load = [&](int64_t t, uint32_t stage) {
        la.load(lds, stage * kStageBytes, wave, k_first + t);
        lb.load(lds, stage * kStageBytes + kTileM * kStepK * 4, wave, k_first + t);
    };
    constexpr int CODES = CODED == kCodedA ? 4 : CODED == kCodedB ? 2 : 1, CODE_STEPS = kCodeK / kStepK;
    uint32_t code[CODES];
    CodeFactor factor[CODES];
    auto load_codes = [&](int64_t step) { // waited for here: a wait in every step would be one for the tiles that are on their way
#pragma unroll
        for (int i = 0; i < CODES; ++i) {
            const int64_t row = (CODED == kCodedA ? m0 + (wave & 1) * 128 : n0 + (wave >> 1) * 64) + 32 * i + (lane & 31), last = (CODED == kCodedA ? M : N) - 1;
            code[i] = codes.p[step / (CODE_STEPS * kCodesAWord) * codes.pitch + (row < last ? row : last)];
        }
#pragma unroll
        for (int i = 0; i < CODES; ++i) asm volatile("" : "+v"(code[i]));
    };
    if (CODED != kPlain && k_steps > 0) load_codes(k_first);
    if (k_steps > 0) load(0, 0);
    if (k_steps > 1) load(1, 1);
    uint32_t now = 0;
    for (int64_t t = 0; t < k_steps; ++t) {
        if (t + 1 < k_steps) stage_barrier<LOADS>();
        else stage_barrier<0>();
        const int64_t step = k_first + t;
        if (CODED != kPlain && t > 0 && step % (CODE_STEPS * kCodesAWord) == 0) load_codes(step);
        if (t + 2 < k_steps) load(t + 2, now == 0 ? 2 : now - 1);
        if (CODED != kPlain && (t == 0 || step % CODE_STEPS == 0))
#pragma unroll
            for (int i = 0; i < CODES; ++i) factor[i].set(code[i], (uint32_t)step / CODE_STEPS % kCodesAWord);
        const char* s = (const char*)lds + now * kStageBytes;
        f16x8 b[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            b[j][0] = rb.read(s, j, 0), b[j][1] = rb.read(s, j, 1);
            if (CODED == kCodedB) b[j][0] = times(times(b[j][0], factor[j % CODES].near), factor[j % CODES].far), b[j][1] = times(b[j][1], factor[j % CODES].low);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f16x8 ah = ra.read(s, i, 0), al = ra.read(s, i, 1);
            if (CODED == kCodedA) ah = times(times(ah, factor[i % CODES].near), factor[i % CODES].far), al = times(al, factor[i % CODES].low);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, b[j][0], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, b[j][1], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, b[j][0], acc[i][j], 0, 0, 0);
            }
        }
        now = now == kStages - 1 ? 0 : now + 1;
    }
}
// acc[i][j][e]: row (wave & 1) * 128 + 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4, column (wave / 2) * 64 + 32 j + lane % 32 of the tile

// Workgroup -> tile.  Workgroups are dealt to the 8 XCDs in turn; each XCD gets a run of tiles of its own, in bands of 8 tile rows
// (column by column inside a band), so that the tiles it works on at a time share rows and columns in its L2.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, int64_t* tm, int64_t* tn) {
    const uint32_t all = tiles_m * tiles_n, per = all / 8, extra = all % 8, xcd = id % 8;
    const uint32_t t = xcd * per + (xcd < extra ? xcd : extra) + id / 8;
    const uint32_t band = t / (8 * tiles_n), first = band * 8, high = tiles_m - first < 8 ? tiles_m - first : 8;
    const uint32_t in = t - first * tiles_n;
    // (the divisions run on the vector units: without this the compiler takes the tile for a per-lane value)
    *tm = __builtin_amdgcn_readfirstlane(first + in % high);
    *tn = __builtin_amdgcn_readfirstlane(in / high);
}

} // namespace tenmo
#endif
