// sample.hip -- the draw of a token under temperature, top-k, top-p and min-p.
//
// With the largest logit m, an entry lies d = log2(e) (m - l) / temperature below it and weighs e = 2^-d.  Entries with
// d >= 44 weigh nothing, on every path: all 2^18 of them together would be below 2^-26 of the largest.
// Weights that are summed in no fixed order (by LDS atomics, over lists) are whole numbers of 2^-44, sums over all entries
// 64-bit floats in a fixed order: a row gives the same token every time.  Entries are ordered by a key, the logit's bits
// turned so that unsigned comparison orders them, and equal keys by index.
//
// One workgroup takes a row and passes over it a few times, from the caches after the first: short loops over vectors in
// flight.  (A row held in registers, 64 logits a thread, was slower: every pass, unrolled over them, is code that runs once
// and has to be fetched.)  The first pass takes the largest logit, and the whole weight where it will be needed.  Filters that
// keep few entries go by a list: the largest logits of the 1,024 threads already hold k entries (or a nucleus' mass), so the
// smallest of those that do bounds the list from below, and what lies above it, a few more than are kept, is ranked entry
// against entry.  Filters that keep many go by a histogram of d, and by the entries of the bin where they end.
//
// It is bound by the vector instructions of a row's passes on its one CU: of 65,536 float32 logits 5 us for the largest and the
// whole weight, 3 for a list; 9 for the histogram, 11 for its bin and the weight before it, 2 to find the draw.  A row without
// filters takes 9.7 us, 40 entries 11.5, a nucleus from a list 13.5, from the histogram 33; 32 rows take as long as one.
#include <algorithm>

#include "clear.hpp"

namespace clear {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kList = 1024, kBins = 1024;
constexpr float kSpan = 44.f, kBinsEach = 22.f;  // d below kSpan; bins of d, the last below kBins
constexpr int kUnit = 44;                         // whole weights are in units of 2^-44: one at least below kSpan
constexpr uint32_t kMostVocab = 1u << 18;         // their sums fit 64 bits
constexpr uint32_t kNever = 0xffffffffu;
constexpr uint32_t kCus = 256;

// 0: never drawn (NaN, -inf); otherwise rising with the logit; 0 and -0 are one
__device__ inline uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    if (!(x > -INFINITY)) return 0;
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }

// floor(e 2^44) of a float in [2^-63, 1]
__device__ inline uint64_t fixed(float e) {
    const uint32_t b = __float_as_uint(e);
    const uint64_t m = (uint64_t)((b & 0x7fffffu) | 0x800000u) << (kUnit - 23);
    return m >> min(127u - (b >> 23), 63u);
}

__device__ inline uint32_t wave_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane((int)x, 63);
}

struct Shared {
    uint64_t bins[kBins];                   // a histogram; with a list: what is kept of each of its entries
    uint64_t order[kList], weight[kList];   // a list: key and flipped index, as one number that falls along the order; weight
    uint64_t order2[kList], weight2[kList]; // of a list's entries those of one bin
    uint64_t part[2][kWaves];               // the waves' sums, of two blocks of sums in turn
    uint64_t extra[kWaves];                 // what the entries of a list add to the waves' parts of the row
    uint64_t above;
    uint32_t listed, listed2, low, bin, found;
};

// Of sixteen values, one a wave: their sums up to each (lane w: up to value w, the same in every row of 16 lanes).
template <class T>
__device__ inline T scan16(T x) {
    x = plus_moved<0x111, 0xf>(x);
    x = plus_moved<0x112, 0xf>(x);
    x = plus_moved<0x114, 0xf>(x);
    return plus_moved<0x118, 0xf>(x);
}

// The sum over the workgroup, in a fixed order.  turn: 0 and 1 in turn, so that one barrier is enough.
template <class T>
__device__ inline T block_sum(T x, Shared& s, int turn) {
    x = wave_sum(x);
    T* part = (T*)s.part[turn];
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
    __syncthreads();
    return from_lane(scan16(part[threadIdx.x % 16]), 15);
}

// The first bin up to which the bins' sum is at least `want` (in s.bin, kNever if there is none) and the sum before it (in
// s.above).  s.bin must be kNever before, with a barrier between; ends with a barrier.
__device__ inline void find_bin(uint64_t want, Shared& s, int turn) {
    const uint64_t mine = s.bins[threadIdx.x], upto = wave_scan(mine);
    if (threadIdx.x % 64 == 63) s.part[turn][threadIdx.x / 64] = upto;
    __syncthreads();
    const uint64_t part = s.part[turn][threadIdx.x % 16];
    const uint64_t before = from_lane(scan16(part) - part, __builtin_amdgcn_readfirstlane(threadIdx.x / 64));
    if (before + upto - mine < want && before + upto >= want) {
        s.bin = threadIdx.x;
        s.above = before + upto - mine;
    }
    __syncthreads();
}

// ---------------------------------------------------------------- a row's logits
// A wave has a contiguous part of the row, taken 64 vectors of 16 bytes at a time; NaN and what lies outside are -inf.
template <class X>
struct Row {
    static constexpr int kVec = 16 / sizeof(X), kStep = 64 * kVec, kFlight = sizeof(X);  // vectors of a thread in flight: 16 logits
    typedef X vec __attribute__((ext_vector_type(kVec)));
    const X* x;        // moved back to a multiple of 16 bytes
    int skip, end;     // the row lies at skip .. end - 1 from there
    int vectors, at0;  // of a thread; its wave's first element
    __device__ Row(const X* row, int vocab) {
        skip = (int)((uintptr_t)row % 16 / sizeof(X));
        x = row - skip;
        end = skip + vocab;
        vectors = (end + kThreads * kVec - 1) / (kThreads * kVec);
        at0 = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * vectors * kStep;
    }
    __device__ int wave_of(uint32_t index) const { return ((int)index + skip) / (vectors * kStep); }
    // f(logits, index): the thread's logits, kFlight vectors at a time; logit e has index + place(e)
    static constexpr int kGroup = kFlight * kVec;
    __device__ static int place(int e) { return e / kVec * kStep + e % kVec; }  // of logit e of a group, from its first
    template <class F>
    __device__ __forceinline__ void groups(F&& f) const {
        const int mine = threadIdx.x % 64 * kVec;
#pragma unroll 1
        for (int j = 0; j < vectors; j += kFlight) {
            const int at = at0 + j * kStep;
            vec v[kFlight];
            if (at >= skip && at + kFlight * kStep <= end && j + kFlight <= vectors) {
#pragma unroll
                for (int u = 0; u < kFlight; u++) v[u] = *(const vec*)(x + at + u * kStep + mine);
            } else {
#pragma unroll
                for (int u = 0; u < kFlight; u++)
#pragma unroll
                    for (int c = 0; c < kVec; c++) {
                        const int i = at + u * kStep + mine + c;
                        v[u][c] = j + u < vectors && i >= skip && i < end ? x[i] : (X)-INFINITY;
                    }
            }
            float one[kGroup];
#pragma unroll
            for (int e = 0; e < kGroup; e++) one[e] = numbered(to_f32((X)v[e / kVec][e % kVec]));
            f(one, at + mine - skip);
        }
    }
    __device__ static float numbered(float x) { return fmaxf(x, -INFINITY); }  // NaN: -inf
    // f(logit, index) for every element of the thread
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        groups([&](const float(&one)[kGroup], int i) {
#pragma unroll
            for (int e = 0; e < kGroup; e++) f(one[e], (uint32_t)(i + place(e)));
        });
    }
};

struct Scale {
    float top, rate;  // log2(e) / temperature, held to where products with it are not NaN
    // how far below the largest, in powers of two
    __device__ float d(float x) const { return fmaxf((top - x) * rate, 0.f); }  // the NaN of inf - inf becomes 0
    __device__ static float e(float d) { return __builtin_amdgcn_exp2f(-d); }
};

// Weights summed.  Those of the largest logit, 1, are counted apart: what the others add to them, which a close
// log-probability hangs on, keeps its float32 bits.
struct Sum {
    double rest = 0.;
    int ones = 0;
    // f(c): the weight of entry c; one(c): whether it is counted
    template <int N, class F, class O>
    __device__ __forceinline__ void add(F&& f, O&& one) {
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < N; c++) {
            const bool is = one(c);
            const float e = f(c);  // computed for all: a select costs less than a branch
            sum += is ? 0.f : e;
            ones += is ? 1 : 0;
        }
        rest += (double)sum;
    }
    __device__ double whole() const { return rest + (double)ones; }
};

// what the filters by rank keep: logits above x, and those that equal it up to index `last`
struct Prefix {
    float x;
    uint32_t last;
    __device__ bool has(float v, uint32_t index) const { return (v > x) | ((v == x) & (index <= last)); }
};

// The first index up to which the weights w(logit, index) >= 0 sum to more than target(their whole sum); mine: the sum over
// the thread's own entries, which s.extra adds to by waves.  Where rounding leaves none, the last one that weighs.  At least
// one weight is above 0.  First the wave whose part it lies in, then all threads on that part, a vector each, and on what
// follows it where the part's entries do not reach the target: sums are rounded, and `mine` may count weights that w does not.
template <class R, class W, class T>
__device__ __forceinline__ uint32_t locate(const R& row, Shared& s, double mine, double& whole, W&& w, T&& target_of) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x % 64;
    // of the waves' sums the first that reaches the target, or the last that weighs; `before`: in, the sum before all of them,
    // out, the sum before that one
    const auto reaching = [&](const double* parts, double target, double& before, bool& reached, double& all) {
        const double part = parts[l % 16], upto = scan16(part);
        const uint32_t over = (uint32_t)__ballot(before + upto > target && part > 0.) & 0xffffu;
        const uint32_t some = (uint32_t)__ballot(part > 0.) & 0xffffu;
        reached = over != 0;
        const int at = over ? __builtin_ctz(over) : some ? 31 - __builtin_clz(some) : 0;
        all = before + from_lane(upto, 15);
        before = at ? before + from_lane(upto, at - 1) : before;
        return some ? at : -1;
    };
    double* part = (double*)s.part[0];
    mine = wave_sum(mine) + (double)s.extra[wave] * 0x1p-44;
    __syncthreads();
    if (l == 0) part[wave] = mine;
    __syncthreads();
    whole = from_lane(scan16(part[l % 16]), 15);
    const double target = target_of(whole);
    double before = 0., all;
    bool reached;
    const int from = max(reaching(part, target, before, reached, all), 0);
    reached = false;
    double* split = (double*)s.part[1];
    const int vectors = (kWaves - from) * row.vectors * 64;  // to the row's end
    for (int v0 = 0; v0 < vectors && !reached; v0 += kThreads) {
        const bool in = v0 + (int)threadIdx.x < vectors;
        const int i = from * row.vectors * R::kStep + (v0 + (int)threadIdx.x) * R::kVec;
        typename R::vec v;
        if (in && i >= row.skip && i + R::kVec <= row.end) v = *(const typename R::vec*)(row.x + i);
        else
#pragma unroll
            for (int c = 0; c < R::kVec; c++) v[c] = in && i + c >= row.skip && i + c < row.end ? row.x[i + c] : -INFINITY;
        float one[R::kVec];
        double vector = 0.;
#pragma unroll
        for (int c = 0; c < R::kVec; c++) {
            one[c] = w(R::numbered(to_f32(v[c])), (uint32_t)(i + c - row.skip));
            vector += (double)one[c];
        }
        const double upto = wave_scan(vector);
        if (l == 63) split[wave] = upto;
        __syncthreads();
        double run = before;
        const int last = reaching(split, target, run, reached, before);
        if (wave == last) {
            const uint64_t over = __ballot(run + upto > target && vector > 0.), some = __ballot(vector > 0.);
            const int lane = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
            if (l == lane) {
                double sum = run + upto - vector;
                bool hit = false;
#pragma unroll
                for (int c = 0; c < R::kVec; c++)
                    if (!hit && one[c] > 0.f) {
                        sum += (double)one[c];
                        hit = sum > target;
                        s.found = (uint32_t)(i + c - row.skip);
                    }
            }
        }
        __syncthreads();
    }
    return s.found;
}

// An entry of a short list against all others: how many come before it and what they weigh.  Some threads share an entry;
// `first` is one of them.
constexpr int kShort = 128;
struct Ranked {
    bool first;
    int rank;
    uint64_t order, weight, before;
};
__device__ inline int sharing(int n) { return n > 64 ? 8 : 16; }
__device__ inline Ranked rank_short(const Shared& s, int n) {
    const int each = sharing(n), i = threadIdx.x / each, sub = threadIdx.x % each;
    Ranked r{i < n && sub == 0, 0, i < n ? s.order[i] : 0, i < n ? s.weight[i] : 0, 0};
    for (int j = sub; j < n; j += each) {
        const uint64_t o = s.order[j], w = s.weight[j];
        if (o > r.order) {
            r.before += w;
            r.rank++;
        }
    }
    for (int m = 1; m < each; m *= 2) {
        r.before += __shfl_xor(r.before, m);
        r.rank += __shfl_xor(r.rank, m);
    }
    return r;
}

// A long list, an entry a thread: the entry up to which the weights sum to at least `want`, 1 <= want <= their sum, in falling
// order (its order is returned).  bin: rises along the order.  A histogram by bin, then the entries of the bin that has it
// against each other.
__device__ inline uint64_t cross(Shared& s, bool in, uint32_t bin, uint64_t order, uint64_t weight, uint64_t want) {
    __syncthreads();
    s.bins[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.bin = kNever, s.listed2 = 0;
    __syncthreads();
    if (in) atomicAdd((unsigned long long*)&s.bins[bin], (unsigned long long)weight);
    __syncthreads();
    find_bin(want, s, 0);
    want -= s.above;
    in = in && bin == s.bin;
    if (in) {
        const uint32_t at = atomicAdd(&s.listed2, 1u);
        s.order2[at] = order;
        s.weight2[at] = weight;
    }
    __syncthreads();
    if (in) {
        uint64_t before = 0;
        for (uint32_t j = 0; j < s.listed2; j++) before += s.order2[j] > order ? s.weight2[j] : 0;
        if (before < want && before + weight >= want) s.above = order;
    }
    __syncthreads();
    return s.above;
}
__device__ inline void add_to_list(Shared& s, float x, uint32_t index, uint64_t weight) {
    const uint32_t at = atomicAdd(&s.listed, 1u);
    if (at < kList) {
        s.order[at] = (uint64_t)key_of(x) << 32 | ~index;
        s.weight[at] = weight;
    }
}

// The shortest prefix of the order, inside `in`, that has `want` entries (by_rank) or whose whole weights sum to at least
// `want`; all of `in` if none does.  Entries with d >= limit must not be needed for it.  A histogram of d gives the bin that
// it ends in; that bin's entries go into a list, or, where they are too many, by the digits of their keys.
// kept: the weight of the thread's entries in the prefix that weigh at least `least`, where s.extra has not got it.
// kInside: whether `in` leaves anything out.
template <bool by_rank, bool kInside, class R>
__device__ __forceinline__ Prefix shortest(const R& row, const Scale& scale, Shared& s, Prefix in, uint64_t want, float limit,
                                           float least, double& kept) {
    const auto inside = [&](float x, uint32_t index) { return !kInside || in.has(x, index); };
    const auto clear = [&] {
        __syncthreads();
        s.bins[threadIdx.x] = 0;
        if (threadIdx.x < kWaves) s.extra[threadIdx.x] = 0;
        if (threadIdx.x == 0) s.bin = kNever, s.listed = 0;
        __syncthreads();
    };
    const auto weigh = [&](const Prefix& p) {
        Sum sum;
        row.groups([&](const float(&x)[R::kGroup], uint32_t i) {
            sum.add<R::kGroup>(
                [&](int c) {
                    const float d = scale.d(x[c]), e = Scale::e(d);
                    return ((d < kSpan) & (e >= least) & p.has(x[c], i + R::place(c))) ? e : 0.f;
                },
                [&](int c) { return (x[c] == scale.top) & p.has(x[c], i + R::place(c)); });
        });
        kept = sum.whole();
    };
    clear();
    row.each([&](float x, uint32_t i) {
        const float d = scale.d(x);
        if ((d < limit) & inside(x, i))
            atomicAdd((unsigned long long*)&s.bins[(int)(d * kBinsEach)], by_rank ? 1ull : (unsigned long long)fixed(Scale::e(d)));
    });
    __syncthreads();
    find_bin(want, s, 0);
    const uint32_t bin = s.bin;
    if (bin == kNever) {
        weigh(in);
        return in;
    }
    want -= s.above;
    {
        const float from = (float)bin, upto = fminf(from + 1.f, limit * kBinsEach);
        Sum sum;
        row.groups([&](const float(&x)[R::kGroup], uint32_t i) {
            uint32_t hits = 0;
            sum.add<R::kGroup>(
                [&](int c) {
                    const float d = scale.d(x[c]), at = d * kBinsEach, e = Scale::e(d);
                    const bool has = inside(x[c], i + R::place(c));
                    hits |= ((at >= from) & (at < upto) & has) ? 1u << c : 0u;
                    return ((at < from) & (e >= least) & has) ? e : 0.f;
                },
                [&](int c) { return (bin > 0) & (x[c] == scale.top) & inside(x[c], i + R::place(c)); });
            while (hits) {  // few
                const int c = __builtin_ctz(hits);
                hits &= hits - 1;
                float v = x[0];
#pragma unroll
                for (int b = 1; b < R::kGroup; b++) v = b == c ? x[b] : v;
                add_to_list(s, v, i + R::place(c), by_rank ? 1ull : fixed(Scale::e(scale.d(v))));
            }
        });
        kept = sum.whole();
    }
    __syncthreads();
    if (s.listed <= kList) {
        const bool there = threadIdx.x < s.listed;
        const uint64_t order = there ? s.order[threadIdx.x] : 0;
        const float d = there ? scale.d(of_key((uint32_t)(order >> 32))) : 0.f, e = Scale::e(d);
        const uint64_t last = cross(s, there, there ? min((uint32_t)((d * kBinsEach - (float)bin) * kBins), kBins - 1u) : 0, order,
                                    there ? s.weight[threadIdx.x] : 0, want);
        if (there && order >= last && e >= least)
            atomicAdd((unsigned long long*)&s.extra[row.wave_of(~(uint32_t)order)], (unsigned long long)fixed(e));
        __syncthreads();
        return Prefix{of_key((uint32_t)(last >> 32)), ~(uint32_t)last};
    }
    uint32_t key = 0;
    uint64_t same = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        clear();
        row.each([&](float x, uint32_t i) {
            const float d = scale.d(x);
            const uint32_t k = key_of(x);
            if (d < limit && (uint32_t)(d * kBinsEach) == bin && (shift == 24 || k >> (shift + 8) == key >> (shift + 8)) &&
                inside(x, i))
                atomicAdd((unsigned long long*)&s.bins[255 - (k >> shift & 255)], by_rank ? 1ull : (unsigned long long)fixed(Scale::e(d)));
        });
        __syncthreads();
        find_bin(want, s, shift / 8 % 2);
        if (s.bin == kNever) {
            weigh(in);
            return in;
        }
        key |= (255 - s.bin) << shift;
        same = s.bins[s.bin];
        want -= s.above;
    }
    const float x = of_key(key);  // the last key; of the entries that have it the first n
    const uint64_t one = by_rank ? 1 : fixed(Scale::e(scale.d(x))), n = (want + one - 1) / one;
    Prefix p{x, x == in.x ? in.last : kNever};
    if (n * one < same) {
        double whole, mine = 0.;
        row.each([&](float v, uint32_t) { mine += v == x ? 1. : 0.; });
        p.last = locate(
            row, s, mine, whole, [&](float v, uint32_t) { return v == x ? 1.f : 0.f; }, [&](double) { return (double)n - 0.5; });
    }
    weigh(p);
    return p;
}

// kWavesEach: waves that a SIMD has to hold.  4, one row on a CU, leaves enough registers; 8 spills 40 and lets two rows
// share a CU: 300 rows of 50,277 by top-k 30.5 against 23.7 us, 256 rows of 65,536 27.9 against 28.8 us.
template <class X, int kWavesEach>
__global__ __launch_bounds__(kThreads, kWavesEach) void k_sample(const X* __restrict__ logits, uint32_t vocab, int64_t stride,
                                                        const float* __restrict__ draws, fhe_ssm_sample_params p,
                                                        int64_t* __restrict__ tokens, float* __restrict__ logprobs) {
    __shared__ Shared s;
    const uint32_t r = blockIdx.x;
    const Row<X> row(logits + (int64_t)r * stride, (int)vocab);
    float temperature = p.temperature ? p.temperature[r] : 1.f;
    int k = p.top_k ? p.top_k[r] : 0;
    const float top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p && p.min_p[r] > 0.f ? fminf(p.min_p[r], 1.f) : 0.f;
    float u = draws[r];
    u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
    if (!(temperature > 0.f)) temperature = 1.f, k = 1;  // the first of the largest
    const bool by_rank = k > 0 && (uint32_t)k < vocab, by_mass = top_p < 1.f;
    const float rate = fminf(fmaxf(1.44269504088896341f / temperature, 1e-30f), 1e30f);

    s.bins[threadIdx.x] = 0;
    if (threadIdx.x < kWaves) s.extra[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.listed = 0, s.low = kNever, s.bin = kNever;

    // the thread's largest logit, and the weight of its entries against it
    float mine = -INFINITY;
    Sum sum;
    const bool weigh = !by_rank && (by_mass || min_p == 0.f);
    if (weigh)
        row.groups([&](const float(&x)[Row<X>::kGroup], int) {
            float most = x[0];
#pragma unroll
            for (int c = 1; c < Row<X>::kGroup; c++) most = fmaxf(most, x[c]);
            if (most > mine) {
                sum.rest = sum.whole() * (double)__builtin_amdgcn_exp2f((mine - most) * rate);
                sum.ones = 0;
                mine = most;
            }
            if (mine > -INFINITY)
                sum.add<Row<X>::kGroup>([&](int c) { return __builtin_amdgcn_exp2f((x[c] - mine) * rate); },
                                        [&](int c) { return x[c] == mine; });
        });
    else row.each([&](float x, uint32_t) { mine = fmaxf(mine, x); });
    const uint32_t key = wave_max(key_of(mine));
    if (threadIdx.x % 64 == 0) s.part[0][threadIdx.x / 64] = key;
    __syncthreads();
    uint32_t most = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) most = max(most, (uint32_t)s.part[0][w]);
    if (!most) {
        if (threadIdx.x == 0) {
            tokens[r] = -1;
            if (logprobs) logprobs[r] = -INFINITY;
        }
        return;
    }
    const Scale scale{of_key(most), rate};
    const float part = fmaxf(top_p, 0.f);
    const auto enough = [&](double whole) { return max((uint64_t)ceil((double)part * whole), (uint64_t)1); };
    // a list of the entries that can be kept, which lie above a bound
    bool listed = false;
    uint64_t want = 0;  // by mass alone: the nucleus' weight
    float low = -INFINITY;
    const float d_mine = scale.d(mine);
    double weight = mine > -INFINITY ? sum.whole() * (double)Scale::e(d_mine) : 0.;
    if (weigh && scale.top == INFINITY) {  // the differences to it were not numbers
        weight = 0.;
        row.each([&](float x, uint32_t) { weight += x == INFINITY ? 1. : 0.; });
    }
    if (by_rank || by_mass) {
        // from the threads' largest: enough of them, or enough weight
        const bool counts = d_mine < kSpan;
        if (!by_rank) want = enough(block_sum(weight, s, 1) * 0x1p44);
        if (counts)
            atomicAdd((unsigned long long*)&s.bins[(int)(d_mine * kBinsEach)], by_rank ? 1ull : (unsigned long long)fixed(Scale::e(d_mine)));
        __syncthreads();
        find_bin(by_rank ? (uint64_t)k : want, s, 0);
        listed = s.bin != kNever;
        if (listed) {
            if (counts && (uint32_t)(d_mine * kBinsEach) <= s.bin) atomicMin(&s.low, key_of(mine));
            __syncthreads();
            low = of_key(s.low);
        }
    } else if (min_p > 0.f) {  // a little below the least weight that min-p keeps
        listed = true;
        low = scale.top - (1.f - __builtin_amdgcn_logf(min_p)) / rate;
    }
    if (listed) {
        row.groups([&](const float(&x)[Row<X>::kGroup], uint32_t i) {
            float most = x[0];
#pragma unroll
            for (int c = 1; c < Row<X>::kGroup; c++) most = fmaxf(most, x[c]);
            if (most >= low) {
#pragma unroll
                for (int c = 0; c < Row<X>::kGroup; c++)
                    if (x[c] >= low) {
                        const float d = scale.d(x[c]);
                        if (d < kSpan) add_to_list(s, x[c], i + Row<X>::place(c), fixed(Scale::e(d)));
                    }
            }
        });
        __syncthreads();
        listed = s.listed <= kList;
    }
    // in 64 bits: a float32 exponent of 10 and more would lose what a close bound on the result can tell
    const auto write = [&](uint32_t token, float x, double rest) {  // rest: what is kept, less the largest
        tokens[r] = token;
        const double off = x >= scale.top ? 0. : ((double)x - (double)scale.top) / (double)temperature;
        if (logprobs) logprobs[r] = (float)(off - log1p(rest));
    };
    if (listed && s.listed <= kShort) {
        const int n = s.listed, each = sharing(n), i = threadIdx.x / each;
        const auto [first, rank, order, weight, before] = rank_short(s, n);
        bool kept = !by_rank || rank < k;
        if (by_mass) {
            if (by_rank) want = enough((double)block_sum(first && kept ? weight : 0, s, 1));
            kept = kept && before < want;
        }
        const float x = of_key((uint32_t)(order >> 32)), e = Scale::e(scale.d(x));
        kept = kept && !(e < min_p);
        if (first) s.bins[i] = kept ? weight : 0;
        const uint64_t whole = block_sum(first && kept ? weight : 0, s, 0);
        const uint64_t target = min((uint64_t)((double)u * (double)whole), whole - 1);
        uint64_t upto = 0;
        const uint32_t flipped = (uint32_t)order;
        for (int j = threadIdx.x % each; j < n; j += each)
            if ((uint32_t)s.order[j] >= flipped) upto += s.bins[j];
        for (int m = 1; m < each; m *= 2) upto += __shfl_xor(upto, m);
        if (first && kept && upto > target && upto - weight <= target) write(~flipped, x, (double)(whole - (1ull << kUnit)) * 0x1p-44);
        return;
    }
    if (listed) {
        const bool there = threadIdx.x < s.listed;
        const uint64_t order = there ? s.order[threadIdx.x] : 0, weight = there ? s.weight[threadIdx.x] : 0;
        const float x = there ? of_key((uint32_t)(order >> 32)) : low, d = scale.d(x), deep = scale.d(low);
        const uint32_t bin = deep > 0.f ? min((uint32_t)(d * ((kBins - 1) / deep)), kBins - 1u) : 0;
        bool kept = there;
        if (by_rank) {  // all threads take part in each of these
            const uint64_t last = cross(s, there, bin, order, 1, (uint64_t)k);
            kept = kept && order >= last;
        }
        if (by_mass) {
            if (by_rank) want = enough((double)block_sum(kept ? weight : 0, s, 1));
            const uint64_t last = cross(s, kept, bin, order, weight, want);
            kept = kept && order >= last;
        }
        kept = kept && !(Scale::e(d) < min_p);
        const uint64_t whole = block_sum(kept ? weight : 0, s, 1);
        const uint64_t target = min((uint64_t)((double)u * (double)whole), whole - 1);
        const uint32_t flipped = (uint32_t)order, index = ~flipped;
        const uint64_t token = cross(s, kept, there ? (uint32_t)((uint64_t)index * kBins / vocab) : 0, flipped, weight, target + 1);
        if (kept && flipped == (uint32_t)token) write(index, x, (double)(whole - (1ull << kUnit)) * 0x1p-44);
        return;
    }

    Prefix keep{-INFINITY, kNever};
    if (by_rank) {
        keep = shortest<true, false>(row, scale, s, keep, (uint64_t)k, kSpan, by_mass ? 0.f : min_p, weight);
        if (by_mass) want = enough((block_sum(weight, s, 1) + from_lane(scan16((double)s.extra[threadIdx.x % 16]), 15) * 0x1p-44) * 0x1p44);
    }
    if (by_mass) {
        // n entries below 1 / n of the weight that may be missing cannot matter: what is above them is enough
        const double missing = ((double)want / part - (double)want) * 0x1p-44;
        float limit = kSpan;
        if (part > 0.f && missing > 0.) limit = fminf(kSpan, 1.f + __builtin_amdgcn_logf((float)((double)vocab / missing)));
        keep = by_rank ? shortest<false, true>(row, scale, s, keep, want, limit, min_p, weight)
                       : shortest<false, false>(row, scale, s, keep, want, limit, min_p, weight);
    }
    if (!weigh && !by_rank && !by_mass)  // min-p alone, with a list that was too long
        row.each([&](float x, uint32_t) {
            const float d = scale.d(x), e = Scale::e(d);
            weight += d < kSpan && e >= min_p ? (double)e : 0.;
        });
    double whole;
    const uint32_t token = locate(
        row, s, weight, whole,
        [&](float x, uint32_t i) {
            const float d = scale.d(x), e = Scale::e(d);
            return d < kSpan && !(e < min_p) && keep.has(x, i) ? e : 0.f;
        },
        [&](double sum) { return (double)u * sum; });
    if (threadIdx.x == 0) write(token, to_f32(logits[(int64_t)r * stride + min(token, vocab - 1)]), whole - 1.);
}

}  // namespace
}  // namespace clear

extern "C" int fhe_ssm_sample(uint32_t type, const void* logits, uint32_t rows, uint32_t vocab, int64_t row_stride,
                              const float* draws, const fhe_ssm_sample_params* params, int64_t* tokens, float* logprobs,
                              void* stream) {
    using namespace clear;
    if (type > FHE_SSM_F16) return fail(CKKS_EINVAL, "sample: unknown type %u", type);
    if (vocab < 1 || vocab > kMostVocab) return fail(CKKS_EINVAL, "sample: a vocabulary of %u is not in [1, %u]", vocab, kMostVocab);
    if (rows > 0x3fffffu) return fail(CKKS_EINVAL, "sample: too many rows");  // a launch has less than 2^32 threads
    if (rows == 0) return CKKS_OK;
    if (!logits || !draws || !params || !tokens) return fail(CKKS_EINVAL, "sample: null argument");
    if (row_stride < 0) return fail(CKKS_EINVAL, "sample: negative stride");
    const auto go = [&](auto t) {
        typedef decltype(t) X;
        const auto kernel = rows <= kCus ? k_sample<X, 4> : k_sample<X, 8>;
        hipLaunchKernelGGL(kernel, dim3(rows), dim3(kThreads), 0, (hipStream_t)stream, (const X*)logits, vocab, row_stride,
                           draws, *params, tokens, logprobs);
    };
    if (type == FHE_SSM_F32) go(0.f);
    else if (type == FHE_SSM_BF16) go(bf16{});
    else go(f16{});
    return launched("sample");
}
