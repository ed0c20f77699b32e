// adamw.hip -- the AdamW step over many tensors at once.
//
//   m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2,  p <- p - lr (decay p + m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps))
//
// Bound by bytes: each entry is read and written once, about 20 vector instructions (8-bit states 60).  82 million entries with bf16
// gradients, 8-bit states and bf16 copies take 264 us, 5.0 TB/s, what a copy reaches; 105 million with states in 32 bits 578,
// 5.1 TB/s; 4.8 million float32 ones without copies, which stay in the last-level cache, 22.7.  Tensors are cut into chunks, a
// workgroup each; a launch takes up to kMostTensors descriptions as its arguments, so that gradients may lie elsewhere at every
// step and nothing has to be laid out on the device.  A workgroup finds its tensor by bisection.
//
// States in 8 bits: m, and the root r of v, whose range is half as wide in powers of two, as floats of 4 exponent and 3
// mantissa bits (a sign, bias 7, the two codes of all ones never made), times a power of two for each 256 entries, the one that
// brings the largest of them into [128, 256).  2^17 below it a magnitude ends.  They are rounded up or down at random, in
// proportion to what is cut off: with b2 near 1 an average that is rounded to nearest would never move.  The random bits are a
// mix of (seed, step, tensor, entry): the same call gives the same result.  An r above 0 is kept above 0, so that m / r stays
// bounded.  A block with a moment that is not finite is NaN from then on (its power is 255), all 256 entries of it; in float32 only
// the entry is lost.  A finite gradient above 1.8e19 has such a moment too, as its square overflows: in float32 its v is infinite
// and the entry moves by its decay alone, in 8 bits, which have no infinity, its block is NaN.
#include <algorithm>
#include <cmath>

#include "rows.hpp"

namespace clear {
namespace {

constexpr uint32_t kMostTensors = 48, kBlock = 256, kChunk = 4096;

struct Tensor {
    float* p;
    const void* g;
    void *m, *v;
    uint8_t* powers;  // [block][2]: m's and r's
    void* copy;
    uint32_t n, first, place;  // entries; its first chunk; its place among all tensors
    float decay;
};
struct Args {
    Tensor tensors[kMostTensors];
    uint32_t count, chunks, each;  // each: entries of a chunk, a multiple of kChunk
    uint32_t copy_type, seed, step;
    float lr, b1, c1, b2, c2, eps;
    float log_b1, log_b2;
    const float *lr_at, *scale_at;
    const int32_t* step_at;
};

__device__ inline uint32_t mixed(uint32_t x) {
    x = (x ^ x >> 16) * 0x9E3779B1u;
    x = (x ^ x >> 15) * 0xB7E15163u;
    return x ^ x >> 16;
}

// What all entries of a step share.
struct Step {
    float lr, first, second, scale;  // first: 1 / (1 - b1^t), second: 1 / sqrt(1 - b2^t)
    uint32_t key;
};

// The largest of the wave's, in all lanes.
__device__ inline uint32_t max64(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, false));
    return max(max(__builtin_amdgcn_readlane((int)x, 0), __builtin_amdgcn_readlane((int)x, 16)),
               max(__builtin_amdgcn_readlane((int)x, 32), __builtin_amdgcn_readlane((int)x, 48)));
}

// the power of two behind a block's codes
__device__ inline float power_of(uint32_t power) {
    return power == 255 ? __builtin_nanf("") : __builtin_ldexpf(1.f, (int)power - 134);
}
// a code's value before that power: exponents 1 to 15 as a float's, 0 as whole steps of 2^-9
__device__ inline float value_of(uint32_t code) {
    const uint32_t low = code & 0x7f;
    const float x = low < 8 ? (float)low * 0x1p-9f : __uint_as_float((low << 20) + (120u << 23));
    return code & 0x80 ? -x : x;
}
// The code of the float with these bits under a power: the magnitude, and what 16 random bits add to it, cut off.
__device__ inline uint32_t code_of(uint32_t bits, uint32_t power, uint32_t draw, bool keep) {
    const uint32_t magnitude = bits & 0x7fffffffu;
    const int up = (int)(magnitude >> 23) - (int)power + 13;  // binades above the lowest whole one
    const int shift = max(-up, 0);
    uint32_t code = 0;
    if (magnitude >= 0x800000u && shift < 12)
        code = ((magnitude & 0x7fffffu) + 0x800000u + (draw << (4 + shift))) >> (20 + shift);
    code += (uint32_t)max(up, 0) * 8 * (code > 0);
    code = min(code, 0x7eu);
    if (keep && magnitude && !code) code = 1;
    return code | (bits >> 31) << 7;
}

// Products and sums of the moments are rounded one by one, so that they come out the same whatever surrounds them.
struct Moments {
    float m, v;
};
__device__ inline Moments moments(const Args& a, float m, float v, float g) {
#pragma clang fp contract(off)
    return {m * a.b1 + g * a.c1, v * a.b2 + (g * g) * a.c2};
}
__device__ inline float moved(const Args& a, const Step& s, float p, float m, float root, float decay) {
    return p - s.lr * (decay * p + (m * s.first) * __builtin_amdgcn_rcpf(root * s.second + a.eps));
}

template <int V>
__device__ inline void write_copy(const Tensor& t, uint32_t type, uint32_t at, const float* p) {
    if (!t.copy) return;
    if (type == FHE_SSM_BF16) store<V>((bf16*)t.copy + at, p);
    else store<V>((f16*)t.copy + at, p);
}

// The root of an average of squares; the instruction takes numbers below the normal ones for 0, and eps may be smaller.
__device__ inline float root_of(float v) {
    const bool low = v < 0x1p-126f;
    const float root = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v);
    return low ? root * 0x1p-32f : root;
}

// V entries of a thread, in 32 bits
template <class G, int V>
__device__ inline void update(const Args& a, const Tensor& t, const Step& s, uint32_t at) {
    float p[V], g[V], m[V], v[V];
    load<V>(t.p + at, p);
    load<V>((const G*)t.g + at, g);
    load<V>((const float*)t.m + at, m);
    load<V>((const float*)t.v + at, v);
#pragma unroll
    for (int c = 0; c < V; c++) {
        const Moments x = moments(a, m[c], v[c], g[c] * s.scale);
        m[c] = x.m, v[c] = x.v;
        p[c] = moved(a, s, p[c], x.m, root_of(x.v), t.decay);
    }
    store<V>(t.p + at, p);
    store<V>((float*)t.m + at, m);
    store<V>((float*)t.v + at, v);
    write_copy<V>(t, a.copy_type, at, p);
}

// A block of 256 entries of a wave, four a lane, in 8 bits.  kWhole: all are there, and vectors may be read.
template <class G, bool kWhole>
__device__ inline void update8(const Args& a, const Tensor& t, const Step& s, uint32_t block, uint32_t lane) {
    const uint32_t at = block * kBlock + lane * 4;
    uint8_t *ms = (uint8_t*)t.m, *rs = (uint8_t*)t.v;
    float p[4], g[4];
    uint32_t mc[4], rc[4];
    if (kWhole) {
        load<4>(t.p + at, p);
        load<4>((const G*)t.g + at, g);
        const uint32_t m4 = *(const uint32_t*)(ms + at), r4 = *(const uint32_t*)(rs + at);
#pragma unroll
        for (int c = 0; c < 4; c++) mc[c] = m4 >> 8 * c & 0xff, rc[c] = r4 >> 8 * c & 0xff;
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const bool in = at + c < t.n;
            p[c] = in ? t.p[at + c] : 0.f;
            g[c] = in ? to_f32(((const G*)t.g)[at + c]) : 0.f;
            mc[c] = in ? ms[at + c] : 0, rc[c] = in ? rs[at + c] : 0;
        }
    }
    const uint32_t powers = *(const uint16_t*)(t.powers + 2 * (size_t)block);
    const float pm = power_of(powers & 0xff), pr = power_of(powers >> 8);
    float m[4], r[4];
    uint32_t most_m = 0, most_v = 0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const float root = value_of(rc[c]) * pr;
        const Moments x = moments(a, value_of(mc[c]) * pm, root * root, g[c] * s.scale);
        m[c] = x.m;
        r[c] = __builtin_sqrtf(x.v);  // to its last bit: what is kept of it follows from the definition alone
        most_m = max(most_m, __float_as_uint(x.m) & 0x7fffffffu);
        most_v = max(most_v, __float_as_uint(x.v) & 0x7fffffffu);
        p[c] = moved(a, s, p[c], x.m, r[c], t.decay);
    }
    const uint32_t field_m = max64(most_m) >> 23, field_v = max64(most_v) >> 23;
    // the root's power from v's, so that its rounding does not decide it
    const bool lost = field_m == 255 || field_v == 255;
    const uint32_t to_m = lost ? 255 : max(field_m, 16u), to_r = lost ? 255 : max((field_v + 127) / 2, 16u);
    uint32_t m4 = 0, r4 = 0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t h = mixed(s.key + at + c);
        mc[c] = lost ? 0 : code_of(__float_as_uint(m[c]), to_m, h & 0xffff, false);
        rc[c] = lost ? 0 : code_of(__float_as_uint(r[c]), to_r, h >> 16, true);
        m4 |= mc[c] << 8 * c, r4 |= rc[c] << 8 * c;
    }
    if (kWhole) {
        store<4>(t.p + at, p);
        *(uint32_t*)(ms + at) = m4;
        *(uint32_t*)(rs + at) = r4;
        write_copy<4>(t, a.copy_type, at, p);
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (at + c < t.n) {
                t.p[at + c] = p[c];
                ms[at + c] = (uint8_t)mc[c], rs[at + c] = (uint8_t)rc[c];
                write_copy<1>(t, a.copy_type, at + c, p + c);
            }
    }
    if (lane == 0) *(uint16_t*)(t.powers + 2 * (size_t)block) = (uint16_t)(to_m | to_r << 8);
}

template <class G, bool k8>
__global__ __launch_bounds__(256) void k_adamw(Args a) {
    uint32_t low = 0, high = a.count;
    while (high - low > 1) {  // the last tensor that begins at this chunk or before
        const uint32_t mid = (low + high) / 2;
        if (a.tensors[mid].first <= blockIdx.x) low = mid;
        else high = mid;
    }
    const Tensor& t = a.tensors[low];
    Step s;
    if (a.step_at && *a.step_at < 1) return;  // 1 - b^0 is 0, and every parameter would be NaN
    const uint32_t step = a.step_at ? (uint32_t)*a.step_at : a.step;
    s.lr = a.lr_at ? *a.lr_at : a.lr;
    s.scale = a.scale_at ? *a.scale_at : 1.f;
    // 1 - b^t = -expm1(t log b), which holds its digits for a b near 1
    s.first = 1.f / -expm1f((float)step * a.log_b1);
    s.second = 1.f / __builtin_sqrtf(-expm1f((float)step * a.log_b2));
    s.key = mixed(a.seed + 0xB7E15163u * step + 0x9E3779B1u * t.place);
    const uint64_t from = (uint64_t)(blockIdx.x - t.first) * a.each;
    const uint32_t upto = (uint32_t)min((uint64_t)t.n, from + a.each);
    constexpr size_t kG = sizeof(G) * 4;
    const bool vectors = ((uintptr_t)t.p % 16 | (uintptr_t)t.g % kG | (uintptr_t)t.m % (k8 ? 4 : 16) |
                          (uintptr_t)t.v % (k8 ? 4 : 16) | (uintptr_t)t.copy % 8) == 0;
    if constexpr (k8) {
        const uint32_t lane = threadIdx.x % 64;
        for (uint32_t b = (uint32_t)(from / kBlock) + threadIdx.x / 64; b * (uint64_t)kBlock < upto; b += 4) {
            if (vectors && (b + 1ull) * kBlock <= upto) update8<G, true>(a, t, s, b, lane);
            else update8<G, false>(a, t, s, b, lane);
        }
    } else {
        uint64_t at = from;
        if (vectors)
#pragma unroll 2
            for (; at + 1024 <= upto; at += 1024) update<G, 4>(a, t, s, (uint32_t)at + threadIdx.x * 4);
        for (at += threadIdx.x; at < upto; at += 256) update<G, 1>(a, t, s, (uint32_t)at);
    }
}

int check(const fhe_ssm_adamw* a, uint32_t count, const fhe_ssm_adamw_tensor* tensors) {
    if (!a || (count && !tensors)) return fail(CKKS_EINVAL, "AdamW: null argument");
    if (a->gradient_type > FHE_SSM_F16) return fail(CKKS_EINVAL, "AdamW: unknown type of gradients %u", a->gradient_type);
    if (a->copy_type != FHE_SSM_BF16 && a->copy_type != FHE_SSM_F16)
        return fail(CKKS_EINVAL, "AdamW: copies are bfloat16 or float16, not of type %u", a->copy_type);
    if (a->state_bits != 8 && a->state_bits != 32) return fail(CKKS_EINVAL, "AdamW: states of %u bits", a->state_bits);
    if (!(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1)) return fail(CKKS_EINVAL, "AdamW: a beta outside [0, 1)");
    if (!(a->eps >= 1e-30f)) return fail(CKKS_EINVAL, "AdamW: eps below 1e-30");  // its reciprocal is a number
    if (!a->step_at && a->step < 1) return fail(CKKS_EINVAL, "AdamW: steps count from 1");
    for (uint32_t i = 0; i < count; i++) {
        const fhe_ssm_adamw_tensor& t = tensors[i];
        if (t.n >= 1ull << 32) return fail(CKKS_EINVAL, "AdamW: tensor %u has 2^32 entries or more", i);
        if (t.n && (!t.param || !t.gradient || !t.first || !t.second || (a->state_bits == 8 && !t.powers)))
            return fail(CKKS_EINVAL, "AdamW: null argument in tensor %u", i);
        if (a->state_bits == 8 && !aligned(t.powers, 2)) return fail(CKKS_EINVAL, "AdamW: powers of tensor %u at an odd address", i);
    }
    return CKKS_OK;
}

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_adamw_step(const fhe_ssm_adamw* a, uint32_t count, const fhe_ssm_adamw_tensor* tensors, void* stream) {
    using namespace clear;
    if (int rc = check(a, count, tensors)) return rc;
    Args k;
    k.copy_type = a->copy_type, k.seed = a->seed, k.step = a->step;
    k.lr = a->lr;
    k.b1 = (float)a->beta1, k.c1 = (float)(1 - a->beta1), k.b2 = (float)a->beta2, k.c2 = (float)(1 - a->beta2);
    k.eps = a->eps;
    k.log_b1 = (float)std::log(a->beta1), k.log_b2 = (float)std::log(a->beta2);
    k.lr_at = a->lr_at, k.scale_at = a->scale_at, k.step_at = a->step_at;
    for (uint32_t at = 0; at < count;) {
        uint64_t total = 0;
        uint32_t next = at;
        for (k.count = 0; next < count && k.count < kMostTensors; next++) {
            const fhe_ssm_adamw_tensor& t = tensors[next];
            if (!t.n) continue;
            k.tensors[k.count++] = {t.param, t.gradient, t.first, t.second, t.powers, t.copy, (uint32_t)t.n, 0, next, t.weight_decay};
            total += t.n;
        }
        at = next;
        if (!k.count) continue;
        // chunks large enough that finding the tensor costs little, and that a launch has some thousands of them
        k.each = kChunk * (uint32_t)std::clamp<uint64_t>(total / (kChunk * 8192ull), 1, 16);
        k.chunks = 0;
        for (uint32_t i = 0; i < k.count; i++) {
            k.tensors[i].first = k.chunks;
            k.chunks += (uint32_t)((k.tensors[i].n + (uint64_t)k.each - 1) / k.each);
        }
        const int rc = by_type(a->gradient_type, [&](auto g) {
            typedef decltype(g) G;
            if (a->state_bits == 8) hipLaunchKernelGGL((k_adamw<G, true>), dim3(k.chunks), dim3(256), 0, (hipStream_t)stream, k);
            else hipLaunchKernelGGL((k_adamw<G, false>), dim3(k.chunks), dim3(256), 0, (hipStream_t)stream, k);
            return launched("AdamW");
        });
        if (rc) return rc;
    }
    return CKKS_OK;
}

}  // extern "C"
