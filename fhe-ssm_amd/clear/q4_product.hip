// q4_product.hip -- rows times a matrix of 4-bit codes with group scales.
//
//   y[r][o] = sum_g s[o][g] ( sum_{j in g} c[o][j] x[r][j]  -  z[o][g] sum_{j in g} x[r][j] )
//
// The products go through 16 x 16 x 32 matrix instructions, 16 weight rows against 16 rows of x, float32 sums.  A code c
// becomes the 16-bit float 16 + c by or-ing its bits into the mantissa of 16.0 (four bits below the leading one: exact in
// bf16 and f16), two codes in an and-or; the 16 is taken out with the zero point, by the group's sum of x, which one more
// matrix instruction with ones gives for all weight rows at once.  bf16 and f16 rows go in as they are; float32 rows go in
// as three bf16 parts (the upper, middle and lower 8 bits of the mantissa, each cut off exactly), so products are exact and
// only the float32 sums round.
#include <algorithm>
#include <type_traits>

#include "clear.hpp"

namespace clear {
namespace {

constexpr uint32_t kRowTile = 16, kBlock = 128;  // weight rows and columns of a stored tile: 64 lanes x 16 bytes

// How a group's scale and zero point of one row are stored: a float16 scale (no zero points), a word of float16 scale and
// float16 16 + zero point, or two float32 of the same.
enum Kind { kHalf, kHalfZero, kFloat };

// the arranged weights: codes [tile][block][lane][4 words], then scales (and zero points) so that what a lane needs lies
// together: [tile][block][16 rows][groups of the block], for groups of a block or more [tile][group][16 rows]
struct Layout {
    uint32_t tiles, blocks, groups, groups_given, each;  // each: groups of a block
    Kind kind;
    size_t scales_at, bytes;
};

Layout layout(const fhe_ssm_q4_matrix& m) {
    Layout y;
    y.tiles = (m.out + kRowTile - 1) / kRowTile;
    y.blocks = (m.in + kBlock - 1) / kBlock;
    y.groups_given = (m.in + m.group - 1) / m.group;
    y.each = m.group < kBlock ? kBlock / m.group : 1;
    y.groups = m.group < kBlock ? y.blocks * y.each : y.groups_given;  // whole blocks of small groups
    y.kind = m.scale_type != FHE_SSM_F16 ? kFloat : m.has_zeros ? kHalfZero : kHalf;
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    y.scales_at = up((size_t)y.tiles * y.blocks * 1024);
    y.bytes = y.scales_at + up((size_t)y.tiles * y.groups * kRowTile * (2u << y.kind));
    return y;
}

// Word j of lane l holds the codes of weight row l % 16, columns 128 block + 32 j + 8 (l / 16) .. + 7: what the lane feeds
// to the block's matrix instruction j.  Codes 2i and 2i + 1 of the eight lie 16 bits apart, at bits 4i and 16 + 4i.
__global__ __launch_bounds__(256) void k_arrange_codes(const uint8_t* __restrict__ codes, int64_t stride, uint32_t out,
                                                       uint32_t in, uint32_t blocks, size_t words,
                                                       uint32_t* __restrict__ to) {
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= words) return;
    const uint32_t j = at % 4, l = at / 4 % 64;
    const size_t tb = at / 256;
    const uint32_t row = (uint32_t)(tb / blocks) * kRowTile + l % 16, col = (uint32_t)(tb % blocks) * kBlock + j * 32 + l / 16 * 8;
    uint32_t w = 0;
    if (row < out) {
        for (uint32_t i = 0; i < 8; i++) {
            if (col + i >= in) break;
            const uint32_t c = codes[(int64_t)row * stride + (col + i) / 2] >> (i % 2 * 4) & 15;
            w |= c << (i / 2 * 4 + i % 2 * 16);
        }
    }
    to[at] = w;
}

template <class S>
__global__ __launch_bounds__(256) void k_arrange_groups(const S* __restrict__ scales, const uint8_t* __restrict__ zeros,
                                                        uint32_t out, uint32_t given, uint32_t groups, uint32_t each,
                                                        Kind kind, size_t n, void* __restrict__ to) {
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= n) return;
    const size_t tb = at / (kRowTile * each);
    const uint32_t row = (uint32_t)(tb / (groups / each)) * kRowTile + at / each % kRowTile;
    const uint32_t g = tb % (groups / each) * each + at % each;
    const bool in = row < out && g < given;
    const float scale = in ? to_f32(scales[(size_t)row * given + g]) : 0.f;
    const float zero = 16.f + (zeros && in ? (float)(zeros[(size_t)row * given + g] & 15) : 8.f);
    if (kind == kFloat) {
        ((float*)to)[2 * at] = scale;
        ((float*)to)[2 * at + 1] = zero;
    } else if (kind == kHalfZero) {
        ((f16*)to)[2 * at] = (f16)scale;
        ((f16*)to)[2 * at + 1] = (f16)zero;
    } else
        ((f16*)to)[at] = (f16)scale;
}

struct Args {
    const u32x4* codes;
    const char* scales;
    const void* x;
    void* y;
    int64_t xs, ys;
    uint32_t out, in, rows, blocks, groups, per_group;  // per_group: blocks of a group, for groups of a block or more
    uint32_t tiles, splits, per_wave, chunk;            // splits of the columns, blocks of one, blocks of one held in LDS
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

// eight elements of a row of x from column k on, zeros past its end, as matrix operands
template <class X>
__device__ inline void load_x(const X* x, uint32_t k, uint32_t in, bool wide, typename Codes<X>::vec (&to)[1]) {
    if (wide && k + 8 <= in) {
        to[0] = *(const typename Codes<X>::vec*)(x + k);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) to[0][i] = k + i < in ? x[k + i] : (X)0.f;
    }
}
__device__ inline void load_x(const float* x, uint32_t k, uint32_t in, bool wide, bf16x8 (&to)[3]) {
    float f[8];
    if (wide && k + 8 <= in) {
        const f32x4 a = *(const f32x4*)(x + k), b = *(const f32x4*)(x + k + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = a[i], f[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = k + i < in ? x[k + i] : 0.f;
    }
    u32x4 part[3];
#pragma unroll
    for (int p = 0; p < 3; p++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t a = __float_as_uint(f[2 * i]), b = __float_as_uint(f[2 * i + 1]);
            part[p][i] = a >> 16 | (b & 0xffff0000u);
            f[2 * i] -= __uint_as_float(a & 0xffff0000u);
            f[2 * i + 1] -= __uint_as_float(b & 0xffff0000u);
        }
#pragma unroll
    for (int p = 0; p < 3; p++) to[p] = __builtin_bit_cast(bf16x8, part[p]);
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

// A workgroup's eight waves take 8 / splits times R tiles of 16 outputs, for 16 C rows of x, and share the columns by `splits`.
// x goes through LDS, as the operands that the matrix instructions take, with each group's sum of x; weights come from memory
// two blocks ahead of their use.  F: groups of a block of 128 columns.
constexpr int kWaves = 8, kAhead = 2;
constexpr uint32_t kLds = 64 << 10, kMostLds = 150 << 10;  // of a workgroup: two a CU, or one where it has to be
template <class X, Kind K, int F, int C, int R>
__global__ __launch_bounds__(64 * kWaves) void k_product(Args a) {
    typedef typename std::conditional<std::is_same<X, f16>::value, f16, bf16>::type E;
    constexpr int P = std::is_same<X, float>::value ? 3 : 1, kFrag = 4 * C * P;  // operands of a block
    typedef typename Codes<E>::vec vec;
    extern __shared__ __attribute__((aligned(16))) char s_bytes[];
    const int l = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t split = wave % a.splits, tiles_at = kWaves / a.splits * R;
    const uint32_t tile0 = blockIdx.x * tiles_at + wave / a.splits * R, row0 = blockIdx.y * (16 * C);
    const uint32_t from = min(split * a.per_wave, a.blocks), to = min(from + a.per_wave, a.blocks);
    vec* s_x = (vec*)s_bytes;                                           // [split][block of the chunk][j][c][p][lane]
    float* s_one = (float*)(s_x + a.splits * a.chunk * kFrag * 64);     // [split][block of the chunk][f][c][row]

    uint32_t mask = Codes<E>::mask, sixteen = Codes<E>::sixteen;
    asm("" : "+s"(mask));
    asm("" : "+v"(sixteen));
    u32x4 w[kAhead][R];
    Groups<K, F> g[kAhead][R];
    // past the end the last block again: a load without a branch needs no wait before it
    const auto load = [&](int slot, uint32_t at) __attribute__((always_inline)) {
        const uint32_t b = min(at, a.blocks - 1);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const uint32_t tile = min(tile0 + r, a.tiles - 1);
            const size_t tb = (size_t)tile * a.blocks + b;
            w[slot][r] = (a.codes + tb * 64)[l];
            const size_t group = F > 1 || a.per_group == 1 ? tb * F : (size_t)tile * a.groups + b / a.per_group;
            g[slot][r].load(a.scales + (group << (K + 1)) * kRowTile + (l / 16 * 4 * F << (K + 1)));
        }
    };
#pragma unroll
    for (int u = 0; u < kAhead; u++) load(u, from + u);

    f32x4 total[R][C];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < C; c++) total[r][c] = f32x4{0, 0, 0, 0};
    for (uint32_t b0 = 0; b0 < a.per_wave; b0 += a.chunk) {
        if (b0) __syncthreads();  // the chunk before has been read
        for (uint32_t e = wave; e < a.splits * a.chunk * C; e += kWaves) {
            const uint32_t c = e % C, sb = e / C, b = sb / a.chunk * a.per_wave + b0 + sb % a.chunk;
            if (b >= a.blocks || b0 + sb % a.chunk >= a.per_wave) continue;
            // lanes past the last row read it again; what they get is not stored
            const X* x = (const X*)a.x + (int64_t)min(row0 + c * 16 + l % 16, a.rows - 1) * a.xs;
            float one[F];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                vec part[P];
                load_x(x, b * kBlock + j * 32 + l / 16 * 8, a.in, a.wide_x, part);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float v = 0.f;
#pragma unroll
                    for (int p = P - 1; p >= 0; p--) v += to_f32((E)part[p][i]);
                    sum += v;
                }
                one[j * F / 4] = j % (4 / F) ? one[j * F / 4] + sum : sum;
#pragma unroll
                for (int p = 0; p < P; p++) s_x[((size_t)sb * kFrag + (j * C + c) * P + p) * 64 + l] = part[p];
            }
#pragma unroll
            for (int f = 0; f < F; f++) {
                one[f] += __shfl_xor(one[f], 16);
                one[f] += __shfl_xor(one[f], 32);
                if (l < 16) s_one[((size_t)sb * F + f) * (16 * C) + c * 16 + l] = K == kHalf ? -24.f * one[f] : one[f];
            }
        }
        __syncthreads();
        const uint32_t end = min(to, from + b0 + a.chunk);
        for (uint32_t b1 = from + b0; b1 < end; b1 += kAhead) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const uint32_t b = b1 + u;
                if (b >= end) break;
                const uint32_t sb = split * a.chunk + (b - from - b0);
#pragma unroll
                for (int f = 0; f < F; f++) {
                    f32x4 sum[R][C];
#pragma unroll
                    for (int c = 0; c < C; c++)
#pragma unroll
                        for (int r = 0; r < R; r++) sum[r][c] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int j = f * (4 / F); j < (f + 1) * (4 / F); j++) {
                        vec part[C][P];
#pragma unroll
                        for (int c = 0; c < C; c++)
#pragma unroll
                            for (int p = 0; p < P; p++) part[c][p] = s_x[((size_t)sb * kFrag + (j * C + c) * P + p) * 64 + l];
#pragma unroll
                        for (int r = 0; r < R; r++) {
                            const vec code = decode<E>(w[u][r][j], mask, sixteen);
#pragma unroll
                            for (int c = 0; c < C; c++)
#pragma unroll
                                for (int p = P - 1; p >= 0; p--) sum[r][c] = Codes<E>::mma(code, part[c][p], sum[r][c]);
                        }
                    }
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        const float one = s_one[((size_t)sb * F + f) * (16 * C) + c * 16 + l % 16];
#pragma unroll
                        for (int r = 0; r < R; r++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                total[r][c][i] = fmaf(g[u][r].scale(i, f),
                                                      K == kHalf ? sum[r][c][i] + one : fmaf(-g[u][r].zero(i, f), one, sum[r][c][i]),
                                                      total[r][c][i]);
                    }
                }
                load(u, b + kAhead);
            }
        }
    }
    const auto store = [&](const f32x4& t, uint32_t tile, int c) __attribute__((always_inline)) {
        const uint32_t row = row0 + c * 16 + l % 16, o = tile * kRowTile + l / 16 * 4;
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
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) store(total[r][c], tile0 + r, c);
        return;
    }
    f32x4* s_part = (f32x4*)s_bytes;  // [tile of the workgroup, c][split][lane]
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < C; c++) s_part[(((wave / a.splits * R + r) * C + c) * a.splits + split) * 64 + l] = total[r][c];
    __syncthreads();
    for (uint32_t e = wave; e < tiles_at * C; e += kWaves) {
        f32x4 t = s_part[e * a.splits * 64 + l];
        for (uint32_t w = 1; w < a.splits; w++) t += s_part[(e * a.splits + w) * 64 + l];
        store(t, blockIdx.x * tiles_at + e / C, e % C);
    }
}

int check(const fhe_ssm_q4_matrix* m) {
    if (!m) return fail(CKKS_EINVAL, "4-bit product: null description");
    if (m->out < 1 || m->in < 1 || m->out > 0x7fffff00u || m->in > 0x7fffff00u)
        return fail(CKKS_EINVAL, "4-bit product: a matrix of %u x %u", m->out, m->in);
    if (m->group != 32 && m->group != 64 && (m->group == 0 || m->group % kBlock))
        return fail(CKKS_EINVAL, "4-bit product: group %u is none of 32, 64 and the multiples of 128", m->group);
    if (m->scale_type > FHE_SSM_F16) return fail(CKKS_EINVAL, "4-bit product: unknown type of scales %u", m->scale_type);
    const Layout y = layout(*m);
    if ((uint64_t)y.tiles * y.blocks > 0x7fffffffull || (uint64_t)y.tiles * y.groups > 0x7fffffffull)
        return fail(CKKS_EINVAL, "4-bit product: the matrix is too large");
    return CKKS_OK;
}

template <class X, Kind K, int F>
int launch_rows(const Args& a, hipStream_t st) {
    constexpr uint32_t P = std::is_same<X, float>::value ? 3 : 1;
    const auto go = [&](auto kernel, uint32_t C, uint32_t R) -> int {
        Args b = a;
        const uint32_t frag = 4096 * C * P + 4 * F * 16 * C;  // of a block in LDS
        b.splits = 1;
        while (b.splits < kWaves && a.tiles / R * b.splits < 2048 && b.splits * 4 <= a.blocks && 2 * b.splits * kAhead * frag <= kMostLds)
            b.splits *= 2;
        b.per_wave = (a.blocks + b.splits - 1) / b.splits;
        b.chunk = std::min(b.per_wave, std::max((uint32_t)kAhead, kLds / (b.splits * frag) / kAhead * kAhead));
        const uint32_t bytes = std::max(b.splits * b.chunk * frag, b.splits > 1 ? kWaves * R * C * 1024 : 0u);
        const uint32_t each = kWaves / b.splits * R;
        const dim3 grid((a.tiles + each - 1) / each, (a.rows + 16 * C - 1) / (16 * C));
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return fail(CKKS_EHIP, "4-bit product: %s", hipGetErrorString(e));
        hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), bytes, st, b);
        return launched("4-bit product");
    };
    if (a.rows <= 16) return go(k_product<X, K, F, 1, 1>, 1, 1);
    if (a.rows <= 32) return go(k_product<X, K, F, 2, 1>, 2, 1);
    return go(k_product<X, K, F, 4, 1>, 4, 1);
}

template <class X, Kind K>
int launch_kind(const Args& a, uint32_t group, hipStream_t st) {
    return group == 32 ? launch_rows<X, K, 4>(a, st) : group == 64 ? launch_rows<X, K, 2>(a, st) : launch_rows<X, K, 1>(a, st);
}

template <class X>
int launch_type(const Args& a, Kind kind, uint32_t group, hipStream_t st) {
    return kind == kHalf ? launch_kind<X, kHalf>(a, group, st)
         : kind == kHalfZero ? launch_kind<X, kHalfZero>(a, group, st)
                             : launch_kind<X, kFloat>(a, group, st);
}

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_q4_bytes(const fhe_ssm_q4_matrix* m, size_t* bytes) {
    if (int rc = clear::check(m)) return rc;
    if (!bytes) return clear::fail(CKKS_EINVAL, "4-bit product: null argument");
    *bytes = clear::layout(*m).bytes;
    return CKKS_OK;
}

int fhe_ssm_q4_arrange(const fhe_ssm_q4_matrix* m, const uint8_t* codes, int64_t code_stride, const void* scales,
                       const uint8_t* zeros, void* weights, void* stream) {
    using namespace clear;
    if (int rc = check(m)) return rc;
    if (!codes || !scales || !weights || !zeros != !m->has_zeros)
        return fail(CKKS_EINVAL, "4-bit product: null argument, or zero points where none are announced");
    if (code_stride < (int64_t)((m->in + 1) / 2)) return fail(CKKS_EINVAL, "4-bit product: rows of codes overlap");
    if (!aligned(weights, 256)) return fail(CKKS_EINVAL, "4-bit product: the arranged weights must lie on 256 bytes");
    const Layout y = layout(*m);
    const hipStream_t st = (hipStream_t)stream;
    uint8_t* to = (uint8_t*)weights;
    const size_t words = (size_t)y.tiles * y.blocks * 256, n = (size_t)y.tiles * y.groups * kRowTile;
    const auto grid = [](size_t k) { return dim3((uint32_t)((k + 255) / 256)); };
    hipLaunchKernelGGL(k_arrange_codes, grid(words), dim3(256), 0, st, codes, code_stride, m->out, m->in, y.blocks, words,
                       (uint32_t*)to);
    const auto put = [&](auto t) {
        typedef decltype(t) S;
        hipLaunchKernelGGL(k_arrange_groups<S>, grid(n), dim3(256), 0, st, (const S*)scales, zeros, m->out, y.groups_given,
                           y.groups, y.each, y.kind, n, (void*)(to + y.scales_at));
    };
    if (m->scale_type == FHE_SSM_F16) put(f16{});
    else if (m->scale_type == FHE_SSM_BF16) put(bf16{});
    else put(0.f);
    return launched("4-bit product: arranging");
}

int fhe_ssm_q4_product(const fhe_ssm_q4_matrix* m, const void* weights, uint32_t type, uint32_t rows, const void* x,
                       int64_t x_stride, void* y, int64_t y_stride, void* stream) {
    using namespace clear;
    if (int rc = check(m)) return rc;
    if (type > FHE_SSM_F16) return fail(CKKS_EINVAL, "4-bit product: unknown type %u", type);
    if (rows == 0) return CKKS_OK;
    if (!weights || !x || !y) return fail(CKKS_EINVAL, "4-bit product: null argument");
    if (!aligned(weights, 256)) return fail(CKKS_EINVAL, "4-bit product: the arranged weights must lie on 256 bytes");
    if (x_stride < 0 || (rows > 1 && y_stride < (int64_t)m->out))
        return fail(CKKS_EINVAL, "4-bit product: rows of y overlap, or a negative stride");
    if (rows > 0x100000) return fail(CKKS_EINVAL, "4-bit product: too many rows");
    const Layout lay = layout(*m);
    const uint8_t* at = (const uint8_t*)weights;
    const size_t size = type_bytes(type);
    const Args a{(const u32x4*)at, (const char*)at + lay.scales_at, x, y, x_stride, y_stride, m->out, m->in, rows, lay.blocks,
                 lay.groups, std::max(1u, m->group / kBlock), lay.tiles, 1, 0, 0,
                 aligned(x, 16) && x_stride * size % 16 == 0, aligned(y, 4 * size) && y_stride % 4 == 0};
    const hipStream_t st = (hipStream_t)stream;
    return type == FHE_SSM_F32 ? launch_type<float>(a, lay.kind, m->group, st)
         : type == FHE_SSM_BF16 ? launch_type<bf16>(a, lay.kind, m->group, st)
                                : launch_type<f16>(a, lay.kind, m->group, st);
}

}  // extern "C"
