// q4_product.hip -- products with 4-bit weights: the layout of the weights and the entry points; the kernel is in
// q4_kernel.hpp, compiled for each type of rows on its own.
#include <algorithm>

#include "q4_kernel.hpp"

namespace clear {
template <>
int launch_q4<float>(const Q4Args&, Kind, uint32_t, hipStream_t);
template <>
int launch_q4<bf16>(const Q4Args&, Kind, uint32_t, hipStream_t);
template <>
int launch_q4<f16>(const Q4Args&, Kind, uint32_t, hipStream_t);

namespace {

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
    y.groups_given = (m.in - 1) / m.group + 1;
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
    if (row < out && col + 8 <= in) {
        uint32_t given;
        __builtin_memcpy(&given, codes + (int64_t)row * stride + col / 2, 4);
        const auto every_other = [](uint32_t c) {
            c &= 0x0f0f0f0fu;
            c = (c | c >> 4) & 0x00ff00ffu;
            return (c | c >> 8) & 0xffffu;
        };
        w = every_other(given) | every_other(given >> 4) << 16;
    } else if (row < out) {
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

int check(const fhe_ssm_q4_matrix* m) {
    if (!m) return fail(CKKS_EINVAL, "4-bit product: null description");
    if (m->out < 1 || m->in < 1 || m->out > 0x7fffff00u || m->in > 0x7fffff00u)
        return fail(CKKS_EINVAL, "4-bit product: a matrix of %u x %u", m->out, m->in);
    if (m->group != 32 && m->group != 64 && (m->group == 0 || m->group % kBlock))
        return fail(CKKS_EINVAL, "4-bit product: group %u is none of 32, 64 and the multiples of 128", m->group);
    if (m->scale_type > FHE_SSM_F16) return fail(CKKS_EINVAL, "4-bit product: unknown type of scales %u", m->scale_type);
    const Layout y = layout(*m);
    if ((uint64_t)y.tiles * y.blocks > 0xffffffull)  // a launch has less than 2^32 threads
        return fail(CKKS_EINVAL, "4-bit product: the matrix is too large");
    return CKKS_OK;
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
    if (code_stride < 0 || (m->out > 1 && code_stride < (int64_t)((m->in + 1) / 2)))
        return fail(CKKS_EINVAL, "4-bit product: rows of codes overlap");
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
    const Q4Args a{(const u32x4*)at, (const char*)at + lay.scales_at, x, y, x_stride, y_stride, m->out, m->in, rows, lay.blocks,
                 lay.groups, std::max(1u, m->group / kBlock), lay.tiles, 1, 0, 0,
                 aligned(x, 16) && x_stride * size % 16 == 0, aligned(y, 4 * size) && y_stride % 4 == 0};
    const hipStream_t st = (hipStream_t)stream;
    return type == FHE_SSM_F32 ? launch_q4<float>(a, lay.kind, m->group, st)
         : type == FHE_SSM_BF16 ? launch_q4<bf16>(a, lay.kind, m->group, st)
                                : launch_q4<f16>(a, lay.kind, m->group, st);
}

}  // extern "C"
