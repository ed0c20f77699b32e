// q4_kernel.hpp -- rows times a matrix of 4-bit codes with group scales: the kernel, and its launch for one type of rows.
//
//   y[r][o] = sum_g s[o][g] ( sum_{j in g} c[o][j] x[r][j]  -  z[o][g] sum_{j in g} x[r][j] )
//
// The products go through 16 x 16 x 32 matrix instructions, 16 weight rows against 16 rows of x, float32 sums.  A code c
// becomes the 16-bit float 16 + c by or-ing its bits into the mantissa of 16.0 (four bits below the leading one: exact in
// bf16 and f16), two codes in an and-or; the 16 is taken out with the zero point, by the group's sum of x.  bf16 and f16 rows
// go in as they are; float32 rows go in as three bf16 parts (the upper, middle and lower 8 bits of the mantissa, each cut off
// exactly), so products are exact and only the float32 sums round.
#pragma once
#include <algorithm>
#include <type_traits>

#include "clear.hpp"

namespace clear {

constexpr uint32_t kRowTile = 16, kBlock = 128;  // weight rows and columns of a stored tile: 64 lanes x 16 bytes

// How a group's scale and zero point of one row are stored: a float16 scale (no zero points), a word of float16 scale and
// float16 16 + zero point, or two float32 of the same.
enum Kind { kHalf, kHalfZero, kFloat };

struct Q4Args {
    const u32x4* codes;
    const char* scales;
    const void* x;
    void* y;
    int64_t xs, ys;
    uint32_t out, in, rows, blocks, groups, per_group;  // per_group: blocks of a group, for groups of a block or more
    uint32_t tiles, splits, per_wave, chunk;            // splits of the columns, blocks of one, those at once in LDS
    bool wide_x, wide_y;
};

// How codes become 16 + c: where their four bits go in a 16-bit float, and what is or-ed in.
template <class E>
struct Codes {  // bf16: 0x4180 | c << 3
    typedef bf16x8 vec;
    static constexpr uint32_t mask = 0x00780078u, sixteen = 0x41804180u;
    static constexpr int shift = 3;
    __device__ static f32x4 mma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Codes<f16> {  // 0x4c00 | c << 6
    typedef f16x8 vec;
    static constexpr uint32_t mask = 0x03c003c0u, sixteen = 0x4c004c00u;
    static constexpr int shift = 6;
    __device__ static f32x4 mma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// mask and sixteen come in registers, one of them vector: an and-or takes one constant
template <class E>
__device__ __forceinline__ typename Codes<E>::vec decode(uint32_t w, uint32_t mask, uint32_t sixteen) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int left = Codes<E>::shift - 4 * i;
        const uint32_t moved = left > 0 ? w << (left > 0 ? left : 0) : w >> (left < 0 ? -left : 0);
        r[i] = (moved & mask) | sixteen;
    }
    return __builtin_bit_cast(typename Codes<E>::vec, r);
}

// eight elements of a row of x from column k on, zeros past its end
template <class X>
struct Eight {
    typedef X vec __attribute__((ext_vector_type(8)));
    vec v;
    __device__ __forceinline__ void load(const X* x, uint32_t k, uint32_t in, bool wide) {
        if (wide && k + 8 <= in) v = *(const vec*)(x + k);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = k + i < in ? x[k + i] : (X)0.f;
    }
};
// as matrix operands: the value itself, or its P upper parts of 8 bits
template <class X, int P>
__device__ __forceinline__ void operands(const Eight<X>& e, typename Codes<X>::vec (&to)[P]) {
    to[0] = e.v;
}
template <int P>
__device__ __forceinline__ void operands(const Eight<float>& e, bf16x8 (&to)[P]) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = e.v[i];
#pragma unroll
    for (int p = 0; p < P; p++) {
        u32x4 part;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t a = __float_as_uint(f[2 * i]), b = __float_as_uint(f[2 * i + 1]);
            part[i] = a >> 16 | (b & 0xffff0000u);
            f[2 * i] -= __uint_as_float(a & 0xffff0000u);
            f[2 * i + 1] -= __uint_as_float(b & 0xffff0000u);
        }
        to[p] = __builtin_bit_cast(bf16x8, part);
    }
}

// Four weight rows' scales and zero points for the F groups of a block, as they are stored.
template <Kind K, int F>
struct Groups {
    uint32_t word[2 * F << K];
    __device__ __forceinline__ void load(const char* at) {
#pragma unroll
        for (int i = 0; i < 2 * F << K; i++) word[i] = ((const uint32_t*)at)[i];
    }
    __device__ __forceinline__ static float half(uint32_t word, int high) {
        return (float)__builtin_bit_cast(f16, (uint16_t)(word >> (16 * high)));
    }
    // of row i in group f: the scale, and 16 + the zero point
    __device__ __forceinline__ float scale(int i, int f) const {
        const int e = i * F + f;
        return K == kHalf ? half(word[e / 2], e % 2) : K == kHalfZero ? half(word[e], 0) : __uint_as_float(word[2 * e % (2 * F << K)]);
    }
    __device__ __forceinline__ float zero(int i, int f) const {
        const int e = i * F + f;
        return K == kHalf ? 24.f : K == kHalfZero ? half(word[e % (2 * F << K)], 1) : __uint_as_float(word[(2 * e + 1) % (2 * F << K)]);
    }
};

// A workgroup's eight waves take 8 / splits tiles of 16 outputs, for 16 C rows of x, and share the columns by `splits`.  x goes
// through LDS in chunks of blocks, as the operands that the matrix instructions take, with each group's sum of x.  Weights
// come from memory A blocks ahead of their use, in a loop without branches: past one the compiler no longer knows how many
// loads are under way, and waits for nearly all of them.  (Six or eight blocks ahead leave room for fewer waves: 16 rows times
// 16,384 x 8,192 21.6 us, 64 rows 67.7 against 52.5; two blocks of x under way while they are laid out, 32 rows of a head
// 14.5 against 11.4: more registers and more code that runs once.)
// It is bound by the weights' way from memory, and for a head by the first and last microseconds of a launch: 65,536 x 768 (27
// MB with scales) 7.6 us for one row, 11.4 for 32; 16,384 x 8,192 (69 MB) 18.7 us for one row, 3.6 TB/s, 22.6 for 16, 52.5 for
// 64, a third of the rate of a large matrix product.
// F: groups of a block of 128 columns.  kPacked: up to five float32 rows, whose three parts are the columns of one tile and are
// summed at the end, instead of three products each (one row of a head 8.9 against 11.3 us).
constexpr int kWaves = 8;
constexpr uint32_t kPackedRows = 5, kCus = 256;
constexpr uint32_t kLds = 64 << 10, kMostLds = 150 << 10;  // of a workgroup: two a CU, or one where it has to be
template <class X, bool kPacked>
constexpr int kProducts = std::is_same<X, float>::value && !kPacked ? 3 : 1;  // of an operand pair
template <class X, bool kPacked>
constexpr int kAheadOf = kProducts<X, kPacked> == 1 ? 4 : 2;  // A
// Sums of a group: of three products the first has one of its own, as its terms are short and their sum, and what the zero
// point takes out of it, hardly round (46 rows of 1,231 columns in groups of 128 are off by 1.8e-7, with one sum by 1.3e-6;
// 64 rows times 4,096 x 4,096 take 37.8 against 34.9 us).
template <class X, bool kPacked>
constexpr int kSums = kProducts<X, kPacked> == 3 ? 2 : 1;

template <class X, Kind K, int F, int C, bool kPacked>
__global__ __launch_bounds__(64 * kWaves) void k_product(Q4Args a) {
    typedef typename std::conditional<std::is_same<X, f16>::value, f16, bf16>::type E;
    constexpr int P = kProducts<X, kPacked>, A = kAheadOf<X, kPacked>, Q = kSums<X, kPacked>, kFrag = 4 * C * P;  // operands of a block
    constexpr int kParts = std::is_same<X, float>::value ? 3 : 1;
    typedef typename Codes<E>::vec vec;
    extern __shared__ __attribute__((aligned(16))) char s_bytes[];
    const int l = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t split = wave % a.splits, tiles_at = kWaves / a.splits, chunk = a.chunk;
    const uint32_t tile = blockIdx.x * tiles_at + wave / a.splits, row0 = blockIdx.y * (16 * C);
    const uint32_t from = min(split * a.per_wave, a.blocks), to = min(from + a.per_wave, a.blocks);
    vec* s_x = (vec*)s_bytes;                                        // [split][block of the chunk][j][c][p][lane]
    float* s_one = (float*)(s_x + a.splits * chunk * kFrag * 64);    // [split][block of the chunk][f][sum][c][row]

    uint32_t mask = Codes<E>::mask, sixteen = Codes<E>::sixteen;
    asm("" : "+s"(mask));
    asm("" : "+v"(sixteen));
    vec ones;
#pragma unroll
    for (int i = 0; i < 8; i++) ones[i] = (E)1.f;
    u32x4 w[A];
    Groups<K, F> g[A];
    const size_t held = min(tile, a.tiles - 1);
    const auto load = [&](int slot, uint32_t at) __attribute__((always_inline)) {
        const uint32_t b = min(at, a.blocks - 1);  // past the end the last block again
        const size_t tb = held * a.blocks + b;
        w[slot] = (a.codes + tb * 64)[l];
        const size_t group = F > 1 || a.per_group == 1 ? tb * F : held * a.groups + b / a.per_group;
        g[slot].load(a.scales + (group << (K + 1)) * kRowTile + (l / 16 * 4 * F << (K + 1)));
    };
#pragma unroll
    for (int u = 0; u < A; u++) load(u, from + u);

    f32x4 total[C];
#pragma unroll
    for (int c = 0; c < C; c++) total[c] = f32x4{0, 0, 0, 0};
    const auto use = [&](int slot, uint32_t sb) __attribute__((always_inline)) {  // sb: the block's place in LDS
#pragma unroll
        for (int f = 0; f < F; f++) {
            f32x4 sum[Q][C];
#pragma unroll
            for (int c = 0; c < Q * C; c++) sum[c / C][c % C] = f32x4{0, 0, 0, 0};
            // all operands of the group are asked for before the first is waited for
            vec x[4 / F][C][P];
#pragma unroll
            for (int j = 0; j < 4 / F; j++)
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int p = 0; p < P; p++) x[j][c][p] = s_x[((size_t)sb * kFrag + ((f * (4 / F) + j) * C + c) * P + p) * 64 + l];
            if constexpr (C * P <= 4) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4 / F; j++) {
                const vec code = decode<E>(w[slot][f * (4 / F) + j], mask, sixteen);
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int p = P - 1; p >= 0; p--) sum[min(p, Q - 1)][c] = Codes<E>::mma(code, x[j][c][p], sum[min(p, Q - 1)][c]);
            }
#pragma unroll
            for (int c = 0; c < C; c++) {
                float one[Q];
#pragma unroll
                for (int n = 0; n < Q; n++) one[n] = s_one[((size_t)sb * F + f) * (16 * C * Q) + (n * C + c) * 16 + l % 16];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float centred = 0.f;
#pragma unroll
                    for (int n = Q - 1; n >= 0; n--) {
                        const float x = K == kHalf ? sum[n][c][i] + one[n] : fmaf(-g[slot].zero(i, f), one[n], sum[n][c][i]);
                        centred = n == Q - 1 ? x : x + centred;
                    }
                    total[c][i] = fmaf(g[slot].scale(i, f), centred, total[c][i]);
                }
            }
        }
    };
    const uint32_t part = kPacked ? min((uint32_t)(l % 16) / a.rows, 2u) : 0;  // of the lane's row
    for (uint32_t b0 = 0; b0 < a.per_wave; b0 += chunk) {
        if (b0) __syncthreads();  // the chunk before has been used
        for (uint32_t e = wave; e < a.splits * chunk * C; e += kWaves) {
            const uint32_t c = e % C, sb = e / C, in_split = b0 + sb % chunk, b = sb / chunk * a.per_wave + in_split;
            if (in_split >= a.per_wave || b >= a.blocks) continue;
            // lanes past the last row read it again; what they get is not stored
            const uint32_t row = kPacked ? min(l % 16 - part * a.rows, a.rows - 1) : min(row0 + c * 16 + l % 16, a.rows - 1);
            const X* x = (const X*)a.x + (int64_t)row * a.xs;
            Eight<X> raw[4];
#pragma unroll
            for (int j = 0; j < 4; j++) raw[j].load(x, b * kBlock + j * 32 + l / 16 * 8, a.in, a.wide_x);
            f32x4 one[Q][F];  // a product with ones sums a row over all lanes that have a part of it
#pragma unroll
            for (int f = 0; f < Q * F; f++) one[f / F][f % F] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                vec parts[kParts], mine[P];
                operands(raw[j], parts);
                if constexpr (kPacked) mine[0] = part == 0 ? parts[0] : part == 1 ? parts[1] : parts[2];
                else
#pragma unroll
                    for (int p = 0; p < P; p++) mine[p] = parts[p];
#pragma unroll
                for (int p = P - 1; p >= 0; p--) one[min(p, Q - 1)][j * F / 4] = Codes<E>::mma(ones, mine[p], one[min(p, Q - 1)][j * F / 4]);
#pragma unroll
                for (int p = 0; p < P; p++) s_x[((size_t)sb * kFrag + (j * C + c) * P + p) * 64 + l] = mine[p];
            }
#pragma unroll
            for (int f = 0; f < F; f++)
#pragma unroll
                for (int n = 0; n < Q; n++)
                    if (l < 16)
                        s_one[((size_t)sb * F + f) * (16 * C * Q) + (n * C + c) * 16 + l] = K == kHalf ? -24.f * one[n][f][0] : one[n][f][0];
        }
        __syncthreads();
        const uint32_t begin = min(from + b0, to), end = min(to, from + b0 + chunk), at = split * chunk;
        uint32_t b = begin;
        for (; b + A <= end; b += A) {
#pragma unroll
            for (int u = 0; u < A; u++) {
                use(u, at + b - begin + u);
                load(u, b + u + A);
            }
        }
#pragma unroll
        for (int u = 0; u < A - 1; u++)  // only behind the last chunk, and the loads with it
            if (b + u < end) use(u, at + b - begin + u);
    }
    const auto store = [&](f32x4 t, uint32_t at, int c) __attribute__((always_inline)) {
        if constexpr (kPacked) {
            f32x4 low, middle;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                low[i] = __shfl(t[i], l + 2 * (int)a.rows);
                middle[i] = __shfl(t[i], l + (int)a.rows);
            }
            t = t + (middle + low);
        }
        const uint32_t row = row0 + c * 16 + l % 16, o = at * kRowTile + l / 16 * 4;
        if (row >= a.rows || o >= a.out) return;
        X* y = (X*)a.y + (int64_t)row * a.ys + o;
        typedef X x4 __attribute__((ext_vector_type(4)));
        if (a.wide_y && o + 4 <= a.out) {
            x4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = from_f32<X>(t[i]);
            *(x4*)y = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (o + i < a.out) y[i] = from_f32<X>(t[i]);
        }
    };
    if (a.splits == 1) {
#pragma unroll
        for (int c = 0; c < C; c++) store(total[c], tile, c);
        return;
    }
    f32x4* s_part = (f32x4*)s_bytes;  // [tile of the workgroup, c][split][lane]
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; c++) s_part[((wave / a.splits * C + c) * a.splits + split) * 64 + l] = total[c];
    __syncthreads();
    for (uint32_t e = wave; e < tiles_at * C; e += kWaves) {
        f32x4 t = s_part[e * a.splits * 64 + l];
        for (uint32_t n = 1; n < a.splits; n++) t += s_part[(e * a.splits + n) * 64 + l];
        store(t, blockIdx.x * tiles_at + e / C, e % C);
    }
}

template <class X, Kind K, int F>
int launch_rows(const Q4Args& a, hipStream_t st) {
    constexpr bool kFloats = std::is_same<X, float>::value;
    const uint32_t row_tiles = (a.rows + 15) / 16;
    const bool packed = kFloats && a.rows <= kPackedRows;
    const uint32_t P = kFloats && !packed ? 3 : 1, A = P == 1 ? 4 : 2;
    const auto frag = [&](uint32_t C) { return C * (4096 * P + 64 * F * (P == 3 ? 2 : 1)); };  // of a block in LDS
    // the columns are split until there are 2,048 waves (16 rows times 16,384 x 8,192: 22.6 us; 1,024 or 4,096 waves: 26.0), as
    // far as A blocks of each split fit the LDS
    const auto splits = [&](uint32_t C) {
        const uint32_t groups = (row_tiles + C - 1) / C;
        uint32_t n = 1;
        while (n < kWaves && (uint64_t)a.tiles * groups * n < 2048 && 2 * n <= a.blocks && 2 * n * A * frag(C) <= kMostLds) n *= 2;
        return n;
    };
    // 16 C rows share a read of the weights; fewer where that alone leaves the GPU empty (64 float32 rows times 4,096 x 4,096:
    // 37.8 against 91.4 us)
    uint32_t C = row_tiles > 2 ? 4 : row_tiles;
    while (C > 1 && (uint64_t)a.tiles * ((row_tiles + C - 1) / C) * splits(C) < 1024) C /= 2;
    const auto go = [&](auto kernel) -> int {
        Q4Args b = a;
        b.splits = splits(C);
        b.per_wave = (a.blocks + b.splits - 1) / b.splits;
        const uint32_t each = kWaves / b.splits;
        const dim3 grid((a.tiles + each - 1) / each, (row_tiles + C - 1) / C);
        const uint32_t room = (uint64_t)grid.x * grid.y <= kCus ? kMostLds : kLds;  // one workgroup a CU, or two (16 rows, 16,384 x 8,192: 22.6, 26.8 us)
        b.chunk = std::min(b.per_wave, std::max(A, room / (b.splits * frag(C)) / A * A));
        const uint32_t bytes = std::max(b.splits * b.chunk * frag(C), b.splits > 1 ? kWaves * C * 1024 : 0u);
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return fail(CKKS_EHIP, "4-bit product: %s", hipGetErrorString(e));
        hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), bytes, st, b);
        return launched("4-bit product");
    };
    if constexpr (kFloats) {
        if (packed) return go(k_product<X, K, F, 1, true>);
    }
    return C == 1 ? go(k_product<X, K, F, 1, false>) : C == 2 ? go(k_product<X, K, F, 2, false>) : go(k_product<X, K, F, 4, false>);
}

template <class X, Kind K>
int launch_kind(const Q4Args& a, uint32_t group, hipStream_t st) {
    return group == 32 ? launch_rows<X, K, 4>(a, st) : group == 64 ? launch_rows<X, K, 2>(a, st) : launch_rows<X, K, 1>(a, st);
}

// one for each type of rows, in a file of its own
template <class X>
int launch_q4(const Q4Args& a, Kind kind, uint32_t group, hipStream_t st);

#define CLEAR_Q4_ROWS(X)                                                                \
    template <>                                                                         \
    int launch_q4<X>(const Q4Args& a, Kind kind, uint32_t group, hipStream_t st) {      \
        return kind == kHalf ? launch_kind<X, kHalf>(a, group, st)                      \
             : kind == kHalfZero ? launch_kind<X, kHalfZero>(a, group, st)              \
                                 : launch_kind<X, kFloat>(a, group, st);                \
    }

}  // namespace clear
