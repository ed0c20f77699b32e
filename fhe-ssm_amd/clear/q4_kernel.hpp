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
    uint32_t tiles, splits, per_wave;                   // splits of the columns, blocks of one
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
// through LDS, as the operands that the matrix instructions take, with each group's sum of x, in chunks: eight units of 128
// columns of 16 rows, U a wave, which wait in the wave's registers while the chunk before them is used.  Weights come from
// memory two blocks ahead of their use.
// F: groups of a block of 128 columns.  kPacked: up to five float32 rows, whose three parts are the columns of one tile and are
// summed at the end, instead of three products each.
constexpr int kWaves = 8, kAhead = 2;
constexpr uint32_t kMostLds = 150 << 10, kPackedRows = 5;
template <class X, Kind K, int F, int C, int U, bool kPacked>
__global__ __launch_bounds__(64 * kWaves) void k_product(Q4Args a) {
    typedef typename std::conditional<std::is_same<X, f16>::value, f16, bf16>::type E;
    constexpr int P = std::is_same<X, float>::value && !kPacked ? 3 : 1, kFrag = 4 * C * P;  // operands of a block
    constexpr int kParts = std::is_same<X, float>::value ? 3 : 1;
    typedef typename Codes<E>::vec vec;
    extern __shared__ __attribute__((aligned(16))) char s_bytes[];
    const int l = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t split = wave % a.splits, tiles_at = kWaves / a.splits, chunk = kWaves * U / (a.splits * C);
    const uint32_t tile = blockIdx.x * tiles_at + wave / a.splits, row0 = blockIdx.y * (16 * C);
    const uint32_t from = min(split * a.per_wave, a.blocks), to = min(from + a.per_wave, a.blocks);
    vec* s_x = (vec*)s_bytes;                                // [split][block of the chunk][j][c][p][lane]
    float* s_one = (float*)(s_x + kWaves * U * 4 * P * 64);  // [split][block of the chunk][f][c][row]

    uint32_t mask = Codes<E>::mask, sixteen = Codes<E>::sixteen;
    asm("" : "+s"(mask));
    asm("" : "+v"(sixteen));
    u32x4 w[kAhead];
    Groups<K, F> g[kAhead];
    const size_t held = min(tile, a.tiles - 1);
    // past the end the last block again: a load without a branch needs no wait before it
    const auto load = [&](int slot, uint32_t at) __attribute__((always_inline)) {
        const uint32_t b = min(at, a.blocks - 1);
        const size_t tb = held * a.blocks + b;
        w[slot] = (a.codes + tb * 64)[l];
        const size_t group = F > 1 || a.per_group == 1 ? tb * F : held * a.groups + b / a.per_group;
        g[slot].load(a.scales + (group << (K + 1)) * kRowTile + (l / 16 * 4 * F << (K + 1)));
    };
    // a wave's units of the chunk at b0: unit u is 16 rows c of a split's block
    Eight<X> raw[U][4];
    const auto unit = [&](int u, uint32_t b0, uint32_t& c, uint32_t& sb, uint32_t& b) __attribute__((always_inline)) {
        const uint32_t e = wave + kWaves * u;
        c = e % C;
        sb = e / C;
        const uint32_t in_split = b0 + sb % chunk;
        b = sb / chunk * a.per_wave + in_split;
        return sb < a.splits * chunk && in_split < a.per_wave && b < a.blocks;
    };
    const uint32_t part = kPacked ? min((uint32_t)(l % 16) / a.rows, 2u) : 0;  // of the lane's row
    const auto fetch = [&](uint32_t b0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint32_t c, sb, b;
            if (!unit(u, b0, c, sb, b)) continue;
            // lanes past the last row read it again; what they get is not stored
            const uint32_t row = kPacked ? min(l % 16 - part * a.rows, a.rows - 1) : min(row0 + c * 16 + l % 16, a.rows - 1);
            const X* x = (const X*)a.x + (int64_t)row * a.xs;
#pragma unroll
            for (int j = 0; j < 4; j++) raw[u][j].load(x, b * kBlock + j * 32 + l / 16 * 8, a.in, a.wide_x);
        }
    };
    fetch(0);
#pragma unroll
    for (int u = 0; u < kAhead; u++) load(u, from + u);

    f32x4 total[C];
#pragma unroll
    for (int c = 0; c < C; c++) total[c] = f32x4{0, 0, 0, 0};
    for (uint32_t b0 = 0; b0 < a.per_wave; b0 += chunk) {
        if (b0) __syncthreads();  // the chunk before has been used
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint32_t c, sb, b;
            if (!unit(u, b0, c, sb, b)) continue;
            float one[F];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                vec parts[kParts], mine[P];
                operands(raw[u][j], parts);
                if constexpr (kPacked) mine[0] = part == 0 ? parts[0] : part == 1 ? parts[1] : parts[2];
                else
#pragma unroll
                    for (int p = 0; p < P; p++) mine[p] = parts[p];
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float v = 0.f;
#pragma unroll
                    for (int p = P - 1; p >= 0; p--) v += to_f32((E)mine[p][i]);
                    sum += v;
                }
                one[j * F / 4] = j % (4 / F) ? one[j * F / 4] + sum : sum;
#pragma unroll
                for (int p = 0; p < P; p++) s_x[((size_t)sb * kFrag + (j * C + c) * P + p) * 64 + l] = mine[p];
            }
#pragma unroll
            for (int f = 0; f < F; f++) {
                one[f] += __shfl_xor(one[f], 16);
                one[f] += __shfl_xor(one[f], 32);
                if (l < 16) s_one[((size_t)sb * F + f) * (16 * C) + c * 16 + l] = K == kHalf ? -24.f * one[f] : one[f];
            }
        }
        __syncthreads();
        if (b0 + chunk < a.per_wave) fetch(b0 + chunk);
        const uint32_t end = min(to, from + b0 + chunk);
        for (uint32_t b1 = from + b0; b1 < end; b1 += kAhead) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const uint32_t b = b1 + u;
                if (b >= end) break;
                const uint32_t sb = split * chunk + (b - from - b0);
#pragma unroll
                for (int f = 0; f < F; f++) {
                    f32x4 sum[C];
#pragma unroll
                    for (int c = 0; c < C; c++) sum[c] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int j = f * (4 / F); j < (f + 1) * (4 / F); j++) {
                        const vec code = decode<E>(w[u][j], mask, sixteen);
#pragma unroll
                        for (int c = 0; c < C; c++)
#pragma unroll
                            for (int p = P - 1; p >= 0; p--)
                                sum[c] = Codes<E>::mma(code, s_x[((size_t)sb * kFrag + (j * C + c) * P + p) * 64 + l], sum[c]);
                    }
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        const float one = s_one[((size_t)sb * F + f) * (16 * C) + c * 16 + l % 16];
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            total[c][i] = fmaf(g[u].scale(i, f), K == kHalf ? sum[c][i] + one : fmaf(-g[u].zero(i, f), one, sum[c][i]),
                                               total[c][i]);
                    }
                }
                load(u, b + kAhead);
            }
        }
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
    constexpr bool kSplit = std::is_same<X, float>::value;  // rows in three parts
    const uint32_t row_tiles = (a.rows + 15) / 16;
    // The columns are split until there are 2,048 waves.  A chunk of one unit a wave has at least two blocks of each split up to
    // splits C = 4; at 8 it takes two units a wave, which three parts have no LDS for.
    const auto splits = [&](uint32_t C, uint32_t most) {
        const uint32_t groups = (row_tiles + C - 1) / C;
        uint32_t n = 1;
        while (a.tiles * groups * n < 2048 && 2 * n <= a.blocks && 2 * n * C <= most) n *= 2;
        return n;
    };
    const bool packed = kSplit && a.rows <= kPackedRows;
    const uint32_t most = kSplit && !packed ? 4 : 8;
    // 16 C rows share a read of the weights; fewer where that alone leaves the GPU empty
    uint32_t C = row_tiles > 2 ? 4 : row_tiles;
    while (C > 1 && a.tiles * ((row_tiles + C - 1) / C) * splits(C, most) < 1024) C /= 2;
    const auto go = [&](auto kernel, uint32_t U, uint32_t P) -> int {
        Q4Args b = a;
        b.splits = splits(C, most);
        b.per_wave = (a.blocks + b.splits - 1) / b.splits;
        const uint32_t tiles = kWaves / b.splits, units = kWaves * U;
        const uint32_t bytes = std::max(units * (4096 * P + 64 * F), b.splits > 1 ? kWaves * C * 1024 : 0u);
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return fail(CKKS_EHIP, "4-bit product: %s", hipGetErrorString(e));
        hipLaunchKernelGGL(kernel, dim3((a.tiles + tiles - 1) / tiles, (row_tiles + C - 1) / C), dim3(64 * kWaves), bytes, st, b);
        return launched("4-bit product");
    };
    const bool two = splits(C, most) * C > 4;
    if constexpr (kSplit) {
        if (packed) return two ? go(k_product<X, K, F, 1, 2, true>, 2, 1) : go(k_product<X, K, F, 1, 1, true>, 1, 1);
        return C == 1 ? go(k_product<X, K, F, 1, 1, false>, 1, 3)
             : C == 2 ? go(k_product<X, K, F, 2, 1, false>, 1, 3)
                      : go(k_product<X, K, F, 4, 1, false>, 1, 3);
    } else {
        if (two)
            return C == 1 ? go(k_product<X, K, F, 1, 2, false>, 2, 1)
                 : C == 2 ? go(k_product<X, K, F, 2, 2, false>, 2, 1)
                          : go(k_product<X, K, F, 4, 2, false>, 2, 1);
        return C == 1 ? go(k_product<X, K, F, 1, 1, false>, 1, 1)
             : C == 2 ? go(k_product<X, K, F, 2, 1, false>, 1, 1)
                      : go(k_product<X, K, F, 4, 1, false>, 1, 1);
    }
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
