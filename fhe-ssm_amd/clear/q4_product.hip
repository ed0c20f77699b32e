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

#include "clear.hpp"

namespace clear {
namespace {

constexpr uint32_t kRowTile = 16, kBlock = 128;  // weight rows and columns of a stored tile: 64 lanes x 16 bytes

// the arranged weights: codes [tile][block][lane][4 words], scales [tile][group][16 rows], zeros [tile][group][16 rows]
struct Layout {
    uint32_t tiles, blocks, groups, groups_given;
    uint32_t scale_bytes;
    size_t scales_at, zeros_at, bytes;
};

Layout layout(const fhe_ssm_q4_matrix& m) {
    Layout y;
    y.tiles = (m.out + kRowTile - 1) / kRowTile;
    y.blocks = (m.in + kBlock - 1) / kBlock;
    y.groups_given = (m.in + m.group - 1) / m.group;
    y.groups = m.group < kBlock ? y.blocks * (kBlock / m.group) : y.groups_given;  // whole blocks of small groups
    y.scale_bytes = m.scale_type == FHE_SSM_F16 ? 2 : 4;
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    y.scales_at = up((size_t)y.tiles * y.blocks * 1024);
    y.zeros_at = y.scales_at + up((size_t)y.tiles * y.groups * kRowTile * y.scale_bytes);
    y.bytes = y.zeros_at + (m.has_zeros ? up((size_t)y.tiles * y.groups * kRowTile) : 0);
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

template <class S, class D>
__global__ __launch_bounds__(256) void k_arrange_groups(const S* __restrict__ from, uint32_t out, uint32_t given,
                                                        uint32_t groups, size_t n, D* __restrict__ to) {
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= n) return;
    const size_t tg = at / kRowTile;
    const uint32_t row = (uint32_t)(tg / groups) * kRowTile + at % kRowTile, g = tg % groups;
    D x = D(0);
    if (row < out && g < given) {
        if constexpr (sizeof(D) == 1) x = from[(size_t)row * given + g] & 15;
        else x = from_f32<D>(to_f32(from[(size_t)row * given + g]));
    }
    to[at] = x;
}

struct Args {
    const u32x4* codes;
    const void* scales;
    const uint8_t* zeros;
    const void* x;
    void* y;
    int64_t xs, ys;
    uint32_t out, in, rows, blocks, groups, per_group;  // per_group: blocks of a group, for groups of a block or more
    uint32_t tiles, per_wave;
    bool half_scales, wide_x, wide_y;
};

// what a code is or-ed into and where its bits go, per pair of codes
template <class F>
struct Codes {  // bf16: 16 + c is 0x4180 | c << 3
    typedef bf16x8 vec;
    static constexpr uint32_t one = 0x3f803f80u;
    __device__ static vec decode(uint32_t w) {
        u32x4 r;
        r.x = (w << 3 & 0x00780078u) | 0x41804180u;
        r.y = (w >> 1 & 0x00780078u) | 0x41804180u;
        r.z = (w >> 5 & 0x00780078u) | 0x41804180u;
        r.w = (w >> 9 & 0x00780078u) | 0x41804180u;
        return __builtin_bit_cast(vec, r);
    }
    __device__ static f32x4 mma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Codes<f16> {  // 16 + c is 0x4c00 | c << 6
    typedef f16x8 vec;
    static constexpr uint32_t one = 0x3c003c00u;
    __device__ static vec decode(uint32_t w) {
        u32x4 r;
        r.x = (w << 6 & 0x03c003c0u) | 0x4c004c00u;
        r.y = (w << 2 & 0x03c003c0u) | 0x4c004c00u;
        r.z = (w >> 2 & 0x03c003c0u) | 0x4c004c00u;
        r.w = (w >> 6 & 0x03c003c0u) | 0x4c004c00u;
        return __builtin_bit_cast(vec, r);
    }
    __device__ static f32x4 mma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

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

// four weight rows' scales and 16 + zero points of a group
__device__ inline void load_group(const Args& a, size_t at, f32x4& s, f32x4& z) {
    if (a.half_scales) {
        typedef f16 f16x4 __attribute__((ext_vector_type(4)));
        const f16x4 h = *(const f16x4*)((const f16*)a.scales + at);
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = (float)h[i];
    } else
        s = *(const f32x4*)((const float*)a.scales + at);
    if (a.zeros) {
        const uint32_t b = *(const uint32_t*)(a.zeros + at);
#pragma unroll
        for (int i = 0; i < 4; i++) z[i] = 16.f + (float)(b >> (8 * i) & 255);
    } else
        z = f32x4{24.f, 24.f, 24.f, 24.f};
}

// A workgroup gives R tiles of 16 outputs for 16 C rows of x; its waves split the columns and join through LDS, in order.
// F: groups of a block of 128 columns.
template <class X, int F, int C, int R>
__global__ __launch_bounds__(512) void k_product(Args a) {
    typedef typename std::conditional<std::is_same<X, f16>::value, f16, bf16>::type E;
    constexpr int P = std::is_same<X, float>::value ? 3 : 1;
    typedef typename Codes<E>::vec vec;
    extern __shared__ f32x4 s_part[];
    const int l = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const uint32_t tile0 = blockIdx.x * R, row0 = blockIdx.y * (16 * C);
    const uint32_t from = wave * a.per_wave, to = min(from + a.per_wave, a.blocks);
    const vec ones = __builtin_bit_cast(vec, u32x4{Codes<E>::one, Codes<E>::one, Codes<E>::one, Codes<E>::one});
    const X* x[C];
#pragma unroll
    for (int c = 0; c < C; c++)  // lanes past the last row read it again; what they get is not stored
        x[c] = (const X*)a.x + (int64_t)min(row0 + c * 16 + l % 16, a.rows - 1) * a.xs;
    f32x4 total[R][C];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < C; c++) total[r][c] = f32x4{0, 0, 0, 0};
    for (uint32_t b = from; b < to; b++) {
        u32x4 w[R];
#pragma unroll
        for (int r = 0; r < R; r++) w[r] = a.codes[((size_t)min(tile0 + r, a.tiles - 1) * a.blocks + b) * 64 + l];
#pragma unroll
        for (int f = 0; f < F; f++) {
            f32x4 sum[R][C], one[C];
#pragma unroll
            for (int c = 0; c < C; c++) {
                one[c] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < R; r++) sum[r][c] = f32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int j = f * (4 / F); j < (f + 1) * (4 / F); j++) {
                vec part[C][P];
#pragma unroll
                for (int c = 0; c < C; c++) {
                    load_x(x[c], b * kBlock + j * 32 + l / 16 * 8, a.in, a.wide_x, part[c]);
#pragma unroll
                    for (int p = P - 1; p >= 0; p--) one[c] = Codes<E>::mma(ones, part[c][p], one[c]);
                }
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const vec code = Codes<E>::decode(w[r][j]);
#pragma unroll
                    for (int c = 0; c < C; c++)
#pragma unroll
                        for (int p = P - 1; p >= 0; p--) sum[r][c] = Codes<E>::mma(code, part[c][p], sum[r][c]);
                }
            }
            const uint32_t g = F > 1 || a.per_group == 1 ? b * F + f : b / a.per_group;
#pragma unroll
            for (int r = 0; r < R; r++) {
                f32x4 s, z;
                load_group(a, ((size_t)min(tile0 + r, a.tiles - 1) * a.groups + g) * kRowTile + l / 16 * 4, s, z);
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) total[r][c][i] = fmaf(s[i], fmaf(-z[i], one[c][i], sum[r][c][i]), total[r][c][i]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < C; c++) s_part[((r * C + c) * waves + wave) * 64 + l] = total[r][c];
    __syncthreads();
    for (int e = wave; e < R * C; e += waves) {
        f32x4 t = s_part[e * waves * 64 + l];
        for (int w = 1; w < waves; w++) t += s_part[(e * waves + w) * 64 + l];
        const uint32_t row = row0 + e % C * 16 + l % 16, o = (tile0 + e / C) * kRowTile + l / 16 * 4;
        if (row >= a.rows) continue;
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

template <class X, int F>
int launch_rows(const Args& a, hipStream_t st) {
    const auto go = [&](auto kernel, uint32_t C, uint32_t R) {
        Args b = a;
        const uint32_t waves = std::min(8u, a.blocks);
        b.per_wave = (a.blocks + waves - 1) / waves;
        const dim3 grid((a.tiles + R - 1) / R, (a.rows + 16 * C - 1) / (16 * C));
        hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), R * C * waves * 1024, st, b);
    };
    if (a.rows <= 16) go(k_product<X, F, 1, 1>, 1, 1);
    else if (a.rows <= 32) go(k_product<X, F, 2, 1>, 2, 1);
    else go(k_product<X, F, 4, 1>, 4, 1);
    return launched("4-bit product");
}

template <class X>
int launch_type(const Args& a, uint32_t group, hipStream_t st) {
    return group == 32 ? launch_rows<X, 4>(a, st) : group == 64 ? launch_rows<X, 2>(a, st) : launch_rows<X, 1>(a, st);
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
    const auto put = [&](auto kernel, const auto* from, auto* into) {
        hipLaunchKernelGGL(kernel, grid(n), dim3(256), 0, st, from, m->out, y.groups_given, y.groups, n, into);
    };
    if (m->scale_type == FHE_SSM_F16) put(k_arrange_groups<f16, f16>, (const f16*)scales, (f16*)(to + y.scales_at));
    else if (m->scale_type == FHE_SSM_BF16) put(k_arrange_groups<bf16, float>, (const bf16*)scales, (float*)(to + y.scales_at));
    else put(k_arrange_groups<float, float>, (const float*)scales, (float*)(to + y.scales_at));
    if (zeros) put(k_arrange_groups<uint8_t, uint8_t>, zeros, to + y.zeros_at);
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
    Args a{(const u32x4*)at, at + lay.scales_at, m->has_zeros ? at + lay.zeros_at : nullptr, x, y, x_stride, y_stride,
           m->out, m->in, rows, lay.blocks, lay.groups, std::max(1u, m->group / kBlock), lay.tiles, 0,
           lay.scale_bytes == 2, aligned(x, 16) && x_stride * size % 16 == 0, aligned(y, 4 * size) && y_stride % 4 == 0};
    const hipStream_t st = (hipStream_t)stream;
    return type == FHE_SSM_F32 ? launch_type<float>(a, m->group, st)
         : type == FHE_SSM_BF16 ? launch_type<bf16>(a, m->group, st)
                                : launch_type<f16>(a, m->group, st);
}

}  // extern "C"
