// sample.hip -- the draw of a token under temperature, top-k, top-p and min-p.
//
// With the largest logit m, an entry weighs e = exp((l - m) / temperature) <= 1, held as a whole number of 2^-44: sums of
// up to 2^18 entries are exact in 64 bits, so they do not depend on their order.  Entries are ordered by a key: the
// logit's bits, turned so that unsigned comparison orders them; equal keys by index.  top-k and top-p each keep a prefix
// of that order, named by the key t of its last entry and the number n of entries of that key in it; the shorter prefix is
// what both keep.
#include <algorithm>

#include "clear.hpp"

namespace clear {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kUnit = 44;              // e is held in units of 2^-44
constexpr uint32_t kMostVocab = 1u << 18;

// 0: never drawn (NaN, -inf); otherwise rising with the logit; 0 and -0 are one
__device__ inline uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    if (!(x > -INFINITY)) return 0;
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }

// floor(e 2^44) of a float in [0, 1]
__device__ inline uint64_t fixed(float e) {
    const uint32_t b = __float_as_uint(e);
    const uint64_t m = (uint64_t)((b & 0x7fffffu) | 0x800000u) << (kUnit - 23);
    return m >> min(127u - (b >> 23), 63u);
}

struct Row {
    float top, rate;  // the largest logit; log2(e) / temperature
    __device__ float e(float x) const {
        return x >= top ? 1.f : exp2f((x - top) * rate);  // the largest also where it is +inf or the rate is
    }
};

__device__ inline uint64_t wave_sum(uint64_t x) {
#pragma unroll
    for (int m = 32; m; m /= 2) x += __shfl_xor(x, m);
    return x;
}

struct Shared {
    uint64_t part[kWaves], mass[256];
    uint32_t count[256];
    uint64_t found[3];
};

__device__ inline uint64_t block_sum(uint64_t x, Shared& s) {
    x = wave_sum(x);
    __syncthreads();
    if (threadIdx.x % 64 == 0) s.part[threadIdx.x / 64] = x;
    __syncthreads();
    uint64_t t = 0;
    for (int w = 0; w < kWaves; w++) t += s.part[w];
    return t;
}

// The prefix of the order that reaches `want` (1 <= want <= the sum over all) when entries count weigh(key): the key of
// its last entry, what lies above that key, by digits of 8 bits from the top.
template <class T, class W>
__device__ inline uint32_t threshold(const T* x, uint32_t vocab, uint64_t want, Shared& s, uint64_t& above, W&& weigh) {
    uint32_t key = 0;
    above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kThreads) s.mass[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
            const float v = to_f32(x[i]);
            const uint32_t k = key_of(v);
            if (k && (shift == 24 || k >> (shift + 8) == key >> (shift + 8)))
                atomicAdd((unsigned long long*)&s.mass[k >> shift & 255], (unsigned long long)weigh(k, v));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint64_t sum = above;
            int d = 255;
            for (; d > 0 && sum + s.mass[d] < want; d--) sum += s.mass[d];
            s.found[0] = d;
            s.found[1] = sum;
        }
        __syncthreads();
        key |= (uint32_t)s.found[0] << shift;
        above = s.found[1];
        __syncthreads();
    }
    return key;
}

// the first index up to which weigh(key, logit, index) sums to at least `want`, or vocab
template <class T, class W>
__device__ inline uint32_t first_reaching(const T* x, uint32_t vocab, uint64_t want, Shared& s, W&& weigh) {
    uint64_t before = 0;
    for (uint32_t i0 = 0; i0 < vocab; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x;
        uint64_t w = 0;
        if (i < vocab) {
            const float v = to_f32(x[i]);
            const uint32_t k = key_of(v);
            if (k) w = weigh(k, v, i);
        }
        const uint64_t sum = block_sum(w, s);
        if (before + sum >= want) {
            uint64_t upto = w;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const uint64_t o = __shfl_up(upto, d);
                if ((int)(threadIdx.x % 64) >= d) upto += o;
            }
            for (int v = 0; v < (int)threadIdx.x / 64; v++) upto += s.part[v];
            upto += before;
            if (upto >= want && upto - w < want) s.found[0] = i;
            __syncthreads();
            return (uint32_t)s.found[0];
        }
        before += sum;
    }
    return vocab;
}

template <class T>
__global__ __launch_bounds__(kThreads) void k_sample(const T* __restrict__ logits, uint32_t vocab, int64_t stride,
                                                     const float* __restrict__ draws, fhe_ssm_sample_params p,
                                                     int64_t* __restrict__ tokens, float* __restrict__ logprobs) {
    __shared__ Shared s;
    const uint32_t r = blockIdx.x;
    const T* x = logits + (int64_t)r * stride;
    float temperature = p.temperature ? p.temperature[r] : 1.f;
    int k = p.top_k ? p.top_k[r] : 0;
    const float top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p && p.min_p[r] > 0.f ? fminf(p.min_p[r], 1.f) : 0.f;
    float u = draws[r];
    u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
    if (!(temperature > 0.f)) temperature = 1.f, k = 1;  // the first of the largest

    uint32_t most = 0;
    uint64_t there = 0;
    for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
        const uint32_t key = key_of(to_f32(x[i]));
        most = max(most, key);
        there += key != 0;
    }
#pragma unroll
    for (int m = 32; m; m /= 2) most = max(most, (uint32_t)__shfl_xor(most, m));
    if (threadIdx.x % 64 == 0) s.part[threadIdx.x / 64] = most;
    __syncthreads();
    for (int w = 0; w < kWaves; w++) most = max(most, (uint32_t)s.part[w]);
    there = block_sum(there, s);
    if (!most) {
        if (threadIdx.x == 0) {
            tokens[r] = -1;
            if (logprobs) logprobs[r] = -INFINITY;
        }
        return;
    }
    const Row row{of_key(most), 1.44269504088896341f / temperature};

    // top-k: the key of the k-th entry and how many of that key are kept
    uint32_t t = 1;
    uint64_t n = ~0ull, above;
    if (k > 0 && (uint64_t)k < there) {
        t = threshold(x, vocab, k, s, above, [](uint32_t, float) { return 1ull; });
        n = k - above;
    }
    // mass of what top-k keeps
    const bool some = n != ~0ull;
    uint64_t mass = 0;
    for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
        const float v = to_f32(x[i]);
        const uint32_t key = key_of(v);
        if (key && (some ? key > t : true)) mass += fixed(row.e(v));
    }
    mass = block_sum(mass, s);
    uint64_t one = some ? fixed(row.e(of_key(t))) : 0;  // each of the entries of key t
    uint64_t total = mass + (some ? n * one : 0);
    if (top_p < 1.f) {
        const uint64_t want = max((uint64_t)ceil((double)max(top_p, 0.f) * (double)total), (uint64_t)1);
        // ties of key t weigh what top-k keeps of them, on the first to come: only their sum matters here
        uint64_t more;
        if (some && want > mass) {  // ends among top-k's last ties
            n = min(n, one ? (want - mass + one - 1) / one : n);
        } else {
            const uint32_t bound = t;
            t = threshold(x, vocab, want, s, more, [&](uint32_t key, float v) -> uint64_t {
                return some && key <= bound ? 0 : fixed(row.e(v));
            });
            one = fixed(row.e(of_key(t)));
            n = one ? (want - more + one - 1) / one : ~0ull;
        }
    }
    const bool cut = t > 1 || n != ~0ull;
    // the last kept index among the entries of key t
    uint32_t last = vocab;
    if (cut && n != ~0ull)
        last = first_reaching(x, vocab, n, s, [&](uint32_t key, float, uint32_t) -> uint64_t { return key == t; });
    const auto weight = [&](uint32_t key, float v, uint32_t i) -> uint64_t {
        if (!(key > t || (key == t && i <= last))) return 0;
        const float e = row.e(v);
        return min_p > 0.f && e < min_p ? 0 : fixed(e);
    };
    uint64_t kept = 0;
    for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
        const float v = to_f32(x[i]);
        const uint32_t key = key_of(v);
        if (key) kept += weight(key, v, i);
    }
    kept = block_sum(kept, s);
    uint64_t want = (uint64_t)((double)u * (double)kept);
    want = min(want, kept - 1) + 1;
    const uint32_t token = min(first_reaching(x, vocab, want, s, weight), vocab - 1);
    if (threadIdx.x == 0) {
        tokens[r] = token;
        if (logprobs) {
            // in 64 bits: a float32 exponent of 10 and more would lose what a close bound on the result can tell
            const float v = to_f32(x[token]);
            const double off = v == row.top ? 0. : ((double)v - (double)row.top) / (double)temperature;
            logprobs[r] = (float)(off - log1p((double)(kept - (1ull << kUnit)) * 0x1p-44));
        }
    }
}

}  // namespace
}  // namespace clear

extern "C" int fhe_ssm_sample(uint32_t type, const void* logits, uint32_t rows, uint32_t vocab, int64_t row_stride,
                              const float* draws, const fhe_ssm_sample_params* params, int64_t* tokens, float* logprobs,
                              void* stream) {
    using namespace clear;
    if (type > FHE_SSM_F16) return fail(CKKS_EINVAL, "sample: unknown type %u", type);
    if (vocab < 1 || vocab > kMostVocab) return fail(CKKS_EINVAL, "sample: a vocabulary of %u is not in [1, %u]", vocab, kMostVocab);
    if (rows > 0x7fffffffu) return fail(CKKS_EINVAL, "sample: too many rows");
    if (rows == 0) return CKKS_OK;
    if (!logits || !draws || !params || !tokens) return fail(CKKS_EINVAL, "sample: null argument");
    if (row_stride < 0) return fail(CKKS_EINVAL, "sample: negative stride");
    const auto go = [&](auto t) {
        hipLaunchKernelGGL(k_sample<decltype(t)>, dim3(rows), dim3(kThreads), 0, (hipStream_t)stream,
                           (const decltype(t)*)logits, vocab, row_stride, draws, *params, tokens, logprobs);
    };
    if (type == FHE_SSM_F32) go(0.f);
    else if (type == FHE_SSM_BF16) go(bf16{});
    else go(f16{});
    return launched("sample");
}
