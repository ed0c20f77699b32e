// token_logprobs.hip -- log-probabilities of given tokens, with entropy and the most likely alternatives, and their gradient.
//
//   with the largest m:  log S = log sum_j exp(l_j - m),  logprob = (l_tok - m) - log S,  p_j = exp((l_j - m) - log S),
//   entropy = log S - sum_j p_j (l_j - m);    d(w logprob + u entropy) / d l_j = w ([j = tok] - p_j) - u p_j (log p_j + entropy)
//
// Differences from the largest, nowhere of large numbers.  A workgroup takes a row and reads it once: a thread holds a
// reference R that is at most kSlack below its largest logit so far, in powers of two and rounded, sum e and sum d e with
// d = l log2(e) - R, e = 2^d, rounded once; when a vector passes R by more, the sums follow it by the difference of the rounded
// ones, and in the end by how far R is from the largest.  That may be 32 powers of two for logits near kHuge; from there on only
// what equals the largest counts.  The threads' sums join in a fixed order.
//
// The alternatives: each strip of a row (the vectors of two neighbouring threads) knows its largest logit and the vector where it
// came first.  The k-th of these in the order of falling logits, then rising index, bounds the k largest from below, and they all
// lie in the k strips that are not behind it: only those are read again, what is not below the bound goes to a list, and the list is
// ranked entry against entry.  Where the list would overflow (large logits that lie together) the row is passed over k times
// for the next largest instead.
//
// Few rows are cut into parts, a workgroup each; a second kernel joins the parts' sums and ranks their alternatives.
//
// Where the weights of the gradient are known the row is read again at once, from the caches, and the gradient written.
// Bound by bytes for many rows: 4,096 bf16 rows of 65,536 with their gradient, read twice and written once, take 236 us, 1.07 GB
// of logits and gradients at 4.5 TB/s (the second reading comes from the caches); about 11 vector instructions a logit, and as many
// for its gradient.  The gradient by itself, where the weights come later, takes 210 us, 5.1 TB/s.  8,192 rows with 20 alternatives
// take 236 us, without 190 (5.7 TB/s); 32 float32 rows with 20 of them 7.1 us and 5.9 for the join.
#include <algorithm>

#include "rows.hpp"

namespace clear {
namespace {

constexpr uint32_t kMostTop = 32, kMostParts = 16, kList = 1024, kWide = 8192, kShortTop = 16;
constexpr uint32_t kEach = 2;  // threads of a strip
constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f;
constexpr float kSlack = 8.f;    // powers of two
// Beside a logit of this size or more every other is 32 or more away and weighs nothing, 2^-46; and below it a rounded reference is
// within 32 powers of two of what it stands for, so that no weight leaves float32's range.
constexpr float kHuge = 0x1p29f;
constexpr int kFlight = 4;  // vectors of a thread on their way

struct Args {
    const void* logits;
    const int64_t* tokens;
    float *logprobs, *entropy, *stats;
    int64_t* top;
    float* top_logprobs;
    const float *weights, *entropy_weights;
    void* grad;
    uint32_t rows, vocab, k;
    int64_t stride, grad_stride;
    // rows in parts of `each` logits
    uint32_t parts, each;
    float* sums;     // [row][part][4]: the part's largest, sum 2^-d, sum d 2^-d
    uint64_t* best;  // [row][part][k]: its largest entries
    float* result;   // [row][4]: the row's largest, log2 S and entropy
};

// 0 for NaN and -inf; otherwise rising with the logit; 0 and -0 are one
__device__ inline uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    if (!(x > -INFINITY)) return 0;
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }

// A row of logits, taken by kThreads threads in vectors of 16 bytes; what lies outside it is -inf.
template <class T, int kThreads>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    const T* x;     // moved back to a multiple of 16 bytes
    int skip, end;  // the row lies at skip .. end - 1 from there
    int vectors;    // of a thread: vector i of thread t is vector i kThreads + t of the row
    __device__ Row(const T* row, uint32_t vocab) {
        skip = (int)((uintptr_t)row % 16 / sizeof(T));
        x = row - skip;
        end = skip + (int)vocab;
        vectors = (end + kThreads * V - 1) / (kThreads * V);
    }
    __device__ void read(int vector, float (&f)[V]) const {
        const int at = vector * V;
        if (at >= skip && at + V <= end) load<V>(x + at, f);
        else
#pragma unroll
            for (int c = 0; c < V; c++) f[c] = at + c >= skip && at + c < end ? to_f32(x[at + c]) : -INFINITY;
    }
    // the thread's vectors first .. first + n - 1; one question for all threads where all are inside the row
    template <int n>
    __device__ void read(int first, float (&f)[n][V]) const {
        const int at = first * kThreads * V;
        if (at >= skip && at + n * kThreads * V <= end)
#pragma unroll
            for (int i = 0; i < n; i++) load<V>(x + at + (i * kThreads + (int)threadIdx.x) * V, f[i]);
        else
#pragma unroll
            for (int i = 0; i < n; i++) read((first + i) * kThreads + (int)threadIdx.x, f[i]);
    }
};

// what is known of a part of a row: its largest, and with d = (m - l) log2(e): sum 2^-d, sum d 2^-d
struct Part {
    float m, s, t;
};
// The parts that 16 or 64 lanes hold, as one, in all of them: all follow the largest, and then it is two sums in a fixed order.
template <int L>
__device__ inline Part joined(Part p) {
    const float m = L == 16 ? max16(p.m) : max64(p.m);
    const float d = p.m == m ? 0.f : (m - p.m) * kLog2e, e = __builtin_amdgcn_exp2f(-d);  // 0 where all are -inf
    const float s = p.s * e, t = p.t * e + (s > 0.f ? d * s : 0.f);
    return {m, L == 16 ? sum16(s) : sum64(s), L == 16 ? sum16(t) : sum64(t)};
}

template <int kThreads>
struct Shared {
    Part part[kThreads / 64];
};
template <int kControl>
__device__ inline uint64_t swapped64(uint64_t x) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), kControl, 0xf, 0xf, false) << 32 |
           (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kControl, 0xf, 0xf, false);
}

template <int kThreads>
struct Alternatives {
    uint64_t best[kThreads / kEach], list[kList + 16], bound, wave[kThreads / 64];
    uint32_t chosen[kMostTop], listed, chosen_count;
};

__device__ inline float log2_p(float x, float m, float log2s) { return __builtin_fmaf(x - m, kLog2e, -log2s); }
__device__ inline float log_p(float x, float m, float log2s) { return __builtin_fmaf(-kLn2, log2s, x - m); }

// An entry's place in the order: its logit's key, then the flipped index; 0 for what is no alternative.
__device__ inline uint64_t entry(float x, uint32_t index) {
    const uint32_t k = key_of(x);
    return k ? (uint64_t)k << 32 | (uint32_t)~index : 0;
}

// Sets the 16 entries behind the list's end to 0, before the barrier that ends its making.
template <int kThreads>
__device__ inline void close_list(Alternatives<kThreads>& s, uint32_t n) {
    if (threadIdx.x < 16) s.list[n + threadIdx.x] = 0;
}

// The k largest entries one by one, to the list.
template <class T, int kThreads>
__device__ void one_by_one(const Row<T, kThreads>& row, uint32_t from, uint32_t k, Alternatives<kThreads>& s) {
    constexpr int V = Row<T, kThreads>::V;
    uint64_t under = ~0ull;
    for (uint32_t i = 0; i < k; i++) {
        uint64_t best = 0;
        for (int j = 0; j < row.vectors; j++) {
            float f[V];
            const int v = j * kThreads + threadIdx.x;
            row.read(v, f);
#pragma unroll
            for (int c = 0; c < V; c++) {
                const uint64_t e = entry(f[c], from + v * V + c - row.skip);
                if (e < under && e > best) best = e;
            }
        }
        for (int o = 32; o > 0; o /= 2) {
            const uint64_t other = __shfl_xor((unsigned long long)best, o);
            best = other > best ? other : best;
        }
        if (threadIdx.x % 64 == 0) s.wave[threadIdx.x / 64] = best;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; w++) best = s.wave[w] > best ? s.wave[w] : best;
        __syncthreads();
        if (threadIdx.x == 0) s.list[i] = best;
        under = best;
    }
    if (threadIdx.x == 0) s.listed = k;
    close_list(s, k);
    __syncthreads();
}

// put(i, entry) for the i-th largest of the list's entries, i < k, and put(i, 0) for what is missing
template <int kThreads, class F>
__device__ void ranked(uint32_t k, const Alternatives<kThreads>& s, F&& put) {
    const uint32_t n = s.listed;
    uint32_t have = n;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t x = s.list[i];
        uint32_t before = 0;
        for (uint32_t j = 0; j < n; j += 16) {  // behind the list's end lie 16 zeros
            uint64_t y[16];
#pragma unroll
            for (int q = 0; q < 16; q++) y[q] = s.list[j + q];
#pragma unroll
            for (int q = 0; q < 16; q++) before += y[q] > x;
        }
        if (x && before < k) put(before, x);
    }
    if (n <= k || s.list[n - 1] == 0) {  // fewer logits than k may be numbers above -inf
        have = 0;
        for (uint32_t j = 0; j < n; j++) have += s.list[j] != 0;
    }
    for (uint32_t i = have + threadIdx.x; i < k; i += kThreads) put(i, 0);
}

// A row's (or its part's, which begins at `from`) k largest to the list, and more; from each thread's largest and the vector
// `first` where it came first.
template <class T, int kThreads>
__device__ void find_alternatives(const Row<T, kThreads>& row, uint32_t from, uint32_t k, float largest, int first,
                                  Alternatives<kThreads>& s) {
    constexpr int V = Row<T, kThreads>::V;
    constexpr uint32_t kStrips = kThreads / kEach;
    // ordered by a vector's first place; the bound takes its last, as the logit itself may lie anywhere in it
    uint64_t mine = entry(largest, (uint32_t)(first * kThreads + (int)threadIdx.x) * V);
    if constexpr (kEach >= 2) mine = max(mine, swapped64<0xb1>(mine));
    if constexpr (kEach == 4) mine = max(mine, swapped64<0x4e>(mine));
    const uint32_t strip = threadIdx.x / kEach, within = threadIdx.x % kEach;
    if (within == 0) s.best[strip] = mine;
    if (threadIdx.x == 0) s.listed = s.chosen_count = 0, s.bound = 0;
    __syncthreads();
    // each of a strip's threads compares it with a share of the others
    uint32_t rank = 0;
#pragma unroll
    for (uint32_t i = 0; i < kStrips / kEach; i++) rank += s.best[i * kEach + within] > mine;
    if constexpr (kEach >= 2) rank += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)rank, 0xb1, 0xf, 0xf, false);
    if constexpr (kEach == 4) rank += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)rank, 0x4e, 0xf, 0xf, false);
    if (mine && rank < k && within == 0) {
        s.chosen[atomicAdd(&s.chosen_count, 1u)] = strip;  // their order says nothing
        if (rank == k - 1) s.bound = mine - (V - 1);
    }
    __syncthreads();
    const uint64_t bound = s.bound;
    const uint32_t per = (uint32_t)row.vectors * kEach, items = s.chosen_count * per;
    for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
        const uint32_t q = i / per, j = i - q * per;
        const int v = (int)(j / kEach * kThreads + s.chosen[q] * kEach + j % kEach);
        float f[V];
        row.read(v, f);
#pragma unroll
        for (int c = 0; c < V; c++) {
            const uint64_t e = entry(f[c], v * V + c);
            if (e && e >= bound) {
                const uint32_t to = atomicAdd(&s.listed, 1u);
                if (to < kList) s.list[to] = e + row.skip - from;  // the flipped index of the row's place
            }
        }
    }
    __syncthreads();
    if (s.listed > kList) return one_by_one(row, from, k, s);
    close_list(s, s.listed);
    __syncthreads();
}

// the token and log-probability of the i-th alternative
__device__ inline void put_alternative(const Args& a, uint32_t r, uint32_t i, uint64_t e, float m, float log2s) {
    a.top[(size_t)r * a.k + i] = e ? (int64_t)(uint32_t)~(uint32_t)e : -1;
    a.top_logprobs[(size_t)r * a.k + i] = e ? log_p(of_key((uint32_t)(e >> 32)), m, log2s) : -INFINITY;
}

// With q = log2 p the gradient is p (-u ln 2 q - (w + u entropy)), and w more at the token.
// The gradient of group `from` of kFlight vectors a thread, of every `step`-th after it.
template <class T, int kThreads>
__device__ void write_gradient(const Args& a, uint32_t r, int64_t token, float m, float log2s, float entropy, int from_group = 0,
                               int step = 1) {
    const T* from = (const T*)a.logits + r * a.stride;
    T* to = (T*)a.grad + r * a.grad_stride;
    const Row<T, kThreads> row(from, a.vocab);
    constexpr int V = Row<T, kThreads>::V;
    const float w = token >= 0 && a.weights ? a.weights[r] : 0.f, u = a.entropy_weights ? a.entropy_weights[r] : 0.f;
    const bool nothing = (w == 0.f && u == 0.f) || (m == -INFINITY && log2s == 0.f);  // whatever the logits are
    const bool same = ((uintptr_t)from ^ (uintptr_t)to) % 16 == 0;
    const int at_token = nothing || token < 0 ? -1 : (int)token + row.skip;
    const float slope = -kLn2 * u, level = -(w + u * entropy);
    to -= row.skip;
    for (int j = from_group * kFlight; j < row.vectors; j += step * kFlight) {
        float f[kFlight][V];
        if (nothing) {
#pragma unroll
            for (int i = 0; i < kFlight; i++)
#pragma unroll
                for (int c = 0; c < V; c++) f[i][c] = 0.f;
        } else {
            row.read(j, f);
#pragma unroll
            for (int i = 0; i < kFlight; i++) {
#pragma unroll
                for (int c = 0; c < V; c++) {
                    const float q = log2_p(f[i][c], m, log2s), p = __builtin_amdgcn_exp2f(q);
                    f[i][c] = p * __builtin_fmaf(__builtin_fmaxf(q, -1e30f), slope, level);  // p of 0 times a q of -inf is 0
                }
                const int at = ((j + i) * kThreads + (int)threadIdx.x) * V;
                if (at_token >= at && at_token < at + V)
#pragma unroll
                    for (int c = 0; c < V; c++) f[i][c] = at + c == at_token ? f[i][c] + w : f[i][c];
            }
        }
        const int begin = j * kThreads * V;
        if (same && begin >= row.skip && begin + kFlight * kThreads * V <= row.end) {
#pragma unroll
            for (int i = 0; i < kFlight; i++) store<V>(to + begin + (i * kThreads + (int)threadIdx.x) * V, f[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kFlight; i++) {
                const int at = begin + (i * kThreads + (int)threadIdx.x) * V;
                if (same && at >= row.skip && at + V <= row.end) store<V>(to + at, f[i]);
                else
#pragma unroll
                    for (int c = 0; c < V; c++)
                        if (at + c >= row.skip && at + c < row.end) to[at + c] = from_f32<T>(f[i][c]);
            }
        }
    }
}

// the token's place, -1 for one that is none
__device__ inline int64_t token_of(const Args& a, uint32_t r) {
    const int64_t token = a.tokens ? a.tokens[r] : -1;
    return token < (int64_t)a.vocab ? token : -1;
}

// a row's numbers from all its logits' sums
struct Numbers {
    float m, log2s, entropy;
    bool none;  // nothing above -inf
    __device__ Numbers(Part p) : m(p.m), none(p.m == -INFINITY && p.s == 0.f) {
        log2s = none ? 0.f : __builtin_amdgcn_logf(p.s);
        entropy = none ? 0.f : kLn2 * (log2s + p.t / p.s);
    }
};
__device__ inline void put_numbers(const Args& a, uint32_t r, int64_t token, float logit, const Numbers& n) {
    if (a.logprobs) a.logprobs[r] = token < 0 ? 0.f : n.none ? -INFINITY : log_p(logit, n.m, n.log2s);
    if (a.entropy) a.entropy[r] = n.entropy;
    if (a.stats) {
        a.stats[2 * (size_t)r] = n.m;
        a.stats[2 * (size_t)r + 1] = n.log2s * kLn2;
    }
}

// a logit as the reference of others: rounded, and not taken into what is done with it
__device__ inline float reference_of(float x) {
#pragma clang fp contract(off)
    return x * kLog2e;
}

// kTop: alternatives are asked for; kGrad: the gradient too, at once; kPart: a row's part, for k_join
template <class T, int kThreads, bool kTop, bool kGrad, bool kPart>
__global__ __launch_bounds__(kThreads) void k_logprobs(Args a) {
    static_assert(!kTop || kThreads <= 256);
    __shared__ Shared<kThreads> s;
    constexpr int V = 16 / sizeof(T);
    const uint32_t r = kPart ? blockIdx.x / a.parts : blockIdx.x, from = kPart ? blockIdx.x % a.parts * a.each : 0;
    const T* logits = (const T*)a.logits + r * a.stride;
    const Row<T, kThreads> row(logits + from, kPart ? min(a.each, a.vocab - from) : a.vocab);
    const int64_t token = kPart ? -1 : token_of(a, r);
    const float given = token < 0 ? 0.f : to_f32(logits[token]);  // asked for before it is needed
    float reference = -INFINITY, largest = -INFINITY, sum = 0.f, along = 0.f;  // the reference times log2(e)
    int first = 0;
    for (int j = 0; j < row.vectors; j += kFlight) {
        float f[kFlight][V];
        row.read(j, f);
#pragma unroll
        for (int i = 0; i < kFlight; i++) {
            float m = f[i][0];
#pragma unroll
            for (int c = 1; c < V; c++) m = __builtin_fmaxf(m, f[i][c]);
            if (!(__builtin_fabsf(m) < kHuge)) {  // masked, or out of all proportion: only what equals the largest counts
                bool bad = false;
#pragma unroll
                for (int c = 0; c < V; c++) bad |= f[i][c] != f[i][c] || f[i][c] == INFINITY;
                // a NaN stays in the sums; what is smaller weighs nothing from here on, what is larger takes the reference along
                if (m > largest) largest = m, first = j + i, reference = __builtin_copysignf(INFINITY, m), sum *= 0.f, along *= 0.f;
                if (m == largest && m > -INFINITY)
#pragma unroll
                    for (int c = 0; c < V; c++) sum += f[i][c] == m ? 1.f : 0.f;
                if (bad) sum = __builtin_nanf("");
                continue;
            }
            if (kTop) first = m > largest ? j + i : first;
            largest = __builtin_fmaxf(largest, m);
            // from one rounded reference to the other, as the summands go by them
            const float next = reference_of(m), above = next - reference;
            if (__builtin_expect(above > kSlack, 0)) {  // rare after the first vectors, and not to be done beside
                const float d = __builtin_fminf(above, 1e6f), e = __builtin_amdgcn_exp2f(-d);
                along = (along - d * sum) * e;
                sum *= e;
                reference = next;
            }
#pragma unroll
            for (int c = 0; c < V; c++) {
                const float d = __builtin_fmaf(f[i][c], kLog2e, -reference), e = __builtin_amdgcn_exp2f(d);
                sum += e;
                along += e * __builtin_fmaxf(d, -1e30f);  // -inf weighs nothing
            }
        }
    }
    Part p{largest, sum, -along};
    if (__builtin_fabsf(largest) < kHuge) {
        const float d = __builtin_fmaf(largest, kLog2e, -reference), e = __builtin_amdgcn_exp2f(-d);
        p.t = (d * sum - along) * e;
        p.s = sum * e;
    }
    p = joined<64>(p);
    if (threadIdx.x % 64 == 0) s.part[threadIdx.x / 64] = p;
    __syncthreads();
    constexpr int kWaves = kThreads / 64;
    p = threadIdx.x % 16 < kWaves ? s.part[threadIdx.x % 16] : Part{-INFINITY, 0.f, 0.f};
    p = joined<16>(p);
    if constexpr (kPart) {
        if (threadIdx.x == 0) {
            float* to = a.sums + (size_t)blockIdx.x * 4;
            to[0] = p.m, to[1] = p.s, to[2] = p.t;
        }
        if constexpr (kTop) {
            __shared__ Alternatives<kThreads> found;
            find_alternatives(row, from, a.k, largest, first, found);
            ranked(a.k, found, [&](uint32_t i, uint64_t e) { a.best[(size_t)blockIdx.x * a.k + i] = e; });
        }
    } else {
        const Numbers n(p);
        if (threadIdx.x == 0) put_numbers(a, r, token, given, n);
        if constexpr (kTop) {
            __shared__ Alternatives<kThreads> found;
            find_alternatives(row, 0, a.k, largest, first, found);
            ranked(a.k, found, [&](uint32_t i, uint64_t e) { put_alternative(a, r, i, e, n.m, n.log2s); });
        }
        if constexpr (kGrad) {
            __syncthreads();  // the gradient may take the logits' place, and their readers are done
            write_gradient<T, kThreads>(a, r, token, n.m, n.log2s, n.entropy);
        }
    }
}

// A row from its parts.
template <class T>
__global__ __launch_bounds__(256) void k_join(Args a) {
    __shared__ Alternatives<256> s;
    // all that is read is asked for at once: a part's sums and last entry by a lane each
    static_assert(kMostParts == 16 && kMostParts * kMostTop <= 512 && 512 <= kList);
    const uint32_t r = blockIdx.x, all = a.parts * a.k, part = threadIdx.x % 16;
    const uint64_t* best = a.best + (size_t)r * all;
    const float* sums = a.sums + ((size_t)r * a.parts + part) * 4;
    const int64_t token = token_of(a, r);
    const float given = token < 0 ? 0.f : to_f32(((const T*)a.logits)[r * a.stride + token]);
    Part p{-INFINITY, 0.f, 0.f};
    if (part < a.parts) p = {sums[0], sums[1], sums[2]};
    uint64_t bound = a.k && part < a.parts ? best[part * a.k + a.k - 1] : 0;
    const uint64_t e0 = threadIdx.x < all ? best[threadIdx.x] : 0, e1 = threadIdx.x + 256 < all ? best[threadIdx.x + 256] : 0;
    if (threadIdx.x == 0) s.listed = 0;
    p = joined<16>(p);
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
        const uint64_t other = __shfl_xor((unsigned long long)bound, o);
        bound = max(bound, other);
    }
    if (a.k) {  // no entry below some part's last is among the row's
        __syncthreads();
        if (e0 && e0 >= bound) s.list[atomicAdd(&s.listed, 1u)] = e0;
        if (e1 && e1 >= bound) s.list[atomicAdd(&s.listed, 1u)] = e1;
        __syncthreads();
        close_list(s, s.listed);
        __syncthreads();
    }
    const Numbers n(p);
    if (threadIdx.x == 0) {
        put_numbers(a, r, token, given, n);
        if (a.grad) {
            float* to = a.result + (size_t)r * 4;
            to[0] = n.m, to[1] = n.log2s, to[2] = n.entropy;
        }
    }
    if (a.k) ranked(a.k, s, [&](uint32_t i, uint64_t e) { put_alternative(a, r, i, e, n.m, n.log2s); });
}

// a row's gradient by itself, `parts` workgroups a row; from the joined parts or from what the caller kept
template <class T, int kThreads>
__global__ __launch_bounds__(kThreads) void k_gradient(Args a) {
    const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const float m = a.result ? a.result[4 * (size_t)r] : a.stats[2 * (size_t)r];
    const float log2s = a.result ? a.result[4 * (size_t)r + 1] : a.stats[2 * (size_t)r + 1] * kLog2e;
    const float entropy = a.result ? a.result[4 * (size_t)r + 2] : a.entropy ? a.entropy[r] : 0.f;
    write_gradient<T, kThreads>(a, r, token_of(a, r), m, log2s, entropy, (int)part, (int)a.parts);
}

int check(const fhe_ssm_token_logprobs* a) {
    if (!a) return fail(CKKS_EINVAL, "token log-probabilities: null description");
    if (a->type > FHE_SSM_F16) return fail(CKKS_EINVAL, "token log-probabilities: unknown type %u", a->type);
    if (a->vocab < 1 || a->vocab > 1u << 18) return fail(CKKS_EINVAL, "token log-probabilities: a vocabulary of %u", a->vocab);
    if (a->top > kMostTop) return fail(CKKS_EINVAL, "token log-probabilities: %u alternatives", a->top);
    if (a->rows >= 1u << 22) return fail(CKKS_EINVAL, "token log-probabilities: too many rows");
    if (a->rows > 1 && a->row_stride < 0) return fail(CKKS_EINVAL, "token log-probabilities: a negative stride");
    return CKKS_OK;
}
int check_gradient(const fhe_ssm_token_logprobs* a, const void* logits, const void* grad) {
    if (a->rows > 1 && a->gradient_stride < (int64_t)a->vocab)
        return fail(CKKS_EINVAL, "token log-probabilities: rows of the gradient overlap");
    if (grad == logits && a->rows > 1 && a->gradient_stride != a->row_stride)
        return fail(CKKS_EINVAL, "token log-probabilities: a gradient in the logits' place has their stride");
    return CKKS_OK;
}
Args args(const fhe_ssm_token_logprobs& a, const void* logits, const int64_t* tokens) {
    Args k{};
    k.logits = logits, k.tokens = tokens, k.rows = a.rows, k.vocab = a.vocab, k.k = a.top;
    k.stride = a.row_stride, k.grad_stride = a.gradient_stride;
    return k;
}
// Rows that a wave reads at once, or where there are many at twice, are a wave's.  (10,000 bf16 rows of 288 with their gradient take
// 21 us, with 256 threads a row 58, of 4,000 40 and 61; of 4,000 with 8 alternatives 31 and 50, but 100 such rows with 16 of them
// 13 and 11.)
template <class T>
bool short_row(const Args& k) {
    return k.vocab <= (k.rows > 1024 ? 2 : 1) * kFlight * 64 * (16 / sizeof(T));
}
// Parts of a row: where rows leave CUs without work, of 4,096 logits at least, two workgroups a CU.  (32 float32 rows of 65,536
// with 20 alternatives take 21 us whole and 13 in parts, 300 bf16 rows of 131,072 with 32 of them 42 and 35.)
void cut(Args& k) {
    k.parts = k.rows < 512 ? std::min({(511 + k.rows) / k.rows, (k.vocab + 4095) / 4096, kMostParts}) : 1;
    k.each = (k.vocab + k.parts - 1) / k.parts;
    k.parts = (k.vocab + k.each - 1) / k.each;
}
size_t workspace_bytes_of(const Args& k) {
    return k.parts > 1 ? (size_t)k.rows * (k.parts * (4 * sizeof(float) + k.k * sizeof(uint64_t)) + 4 * sizeof(float)) : 0;
}

template <class T, int kThreads>
int run_gradient(const Args& k, hipStream_t st) {
    hipLaunchKernelGGL((k_gradient<T, kThreads>), dim3(k.rows * k.parts), dim3(kThreads), 0, st, k);
    return launched("token log-probabilities: gradient");
}

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_token_logprobs_workspace(const fhe_ssm_token_logprobs* a, size_t* bytes) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (!bytes) return fail(CKKS_EINVAL, "token log-probabilities: null argument");
    Args k{};
    k.rows = a->rows, k.vocab = a->vocab, k.k = a->top;
    if (k.rows) cut(k);
    *bytes = workspace_bytes_of(k);
    return CKKS_OK;
}

int fhe_ssm_token_logprobs_forward(const fhe_ssm_token_logprobs* a, const void* logits, const int64_t* tokens,
                                   float* logprobs, float* entropy, float* statistics, int64_t* top, float* top_logprobs,
                                   const float* weights, const float* entropy_weights, void* gradient, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->rows == 0) return CKKS_OK;
    if (!logits || (logprobs && !tokens) || (a->top && (!top || !top_logprobs)) || (weights && !tokens))
        return fail(CKKS_EINVAL, "token log-probabilities: null argument");
    if (gradient)
        if (int rc = check_gradient(a, logits, gradient)) return rc;
    Args k = args(*a, logits, tokens);
    k.logprobs = logprobs, k.entropy = entropy, k.stats = statistics, k.top = top, k.top_logprobs = top_logprobs;
    k.weights = weights, k.entropy_weights = entropy_weights, k.grad = gradient;
    cut(k);
    if (const size_t need = workspace_bytes_of(k)) {
        if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
            return fail(CKKS_EINVAL, "token log-probabilities: the workspace must have %zu bytes and lie on 16", need);
        k.result = (float*)workspace;
        k.sums = k.result + 4 * (size_t)k.rows;
        k.best = (uint64_t*)(k.sums + 4 * (size_t)k.rows * k.parts);
    }
    const hipStream_t st = (hipStream_t)stream;
    return by_type(a->type, [&](auto t) {
        typedef decltype(t) T;
        const auto run = [&](auto n, auto top, auto grad, auto part) {
            constexpr int kThreads = decltype(n)::value;
            hipLaunchKernelGGL((k_logprobs<T, kThreads, decltype(top)::value, decltype(grad)::value, decltype(part)::value>),
                               dim3(k.rows * k.parts), dim3(kThreads), 0, st, k);
            return launched("token log-probabilities");
        };
        const std::true_type yes;
        const std::false_type no;
        const std::integral_constant<int, 64> wave;
        const std::integral_constant<int, 256> few;
        const std::integral_constant<int, 1024> many;
        if (k.parts > 1) {
            if (int rc = k.k ? run(few, yes, no, yes) : run(few, no, no, yes)) return rc;
            hipLaunchKernelGGL(k_join<T>, dim3(k.rows), dim3(256), 0, st, k);
            if (int rc = launched("token log-probabilities: join")) return rc;
            return k.grad ? run_gradient<T, 256>(k, st) : (int)CKKS_OK;
        }
        if (k.k) {
            // a wave has half as many strips as threads: with 32 alternatives all of them would be read again
            if (short_row<T>(k) && k.k <= kShortTop) return k.grad ? run(wave, yes, yes, no) : run(wave, yes, no, no);
            return k.grad ? run(few, yes, yes, no) : run(few, yes, no, no);
        }
        if (short_row<T>(k)) return k.grad ? run(wave, no, yes, no) : run(wave, no, no, no);
        // A long row has a whole CU's threads, so that what lies between its two readings stays in the caches: 4,096 rows of
        // 65,536 in bf16 take 236 us with their gradient, with 256 threads a row 288.
        if (k.vocab > kWide) return k.grad ? run(many, no, yes, no) : run(many, no, no, no);
        return k.grad ? run(few, no, yes, no) : run(few, no, no, no);
    });
}

int fhe_ssm_token_logprobs_gradient(const fhe_ssm_token_logprobs* a, const void* logits, const int64_t* tokens,
                                    const float* statistics, const float* entropy, const float* weights, const float* entropy_weights,
                                    void* gradient, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->rows == 0) return CKKS_OK;
    if (!logits || !statistics || !gradient || (weights && !tokens) || (entropy_weights && !entropy))
        return fail(CKKS_EINVAL, "token log-probabilities: null argument");
    if (int rc = check_gradient(a, logits, gradient)) return rc;
    Args k = args(*a, logits, tokens);
    k.stats = (float*)statistics, k.entropy = (float*)entropy, k.weights = weights, k.entropy_weights = entropy_weights, k.grad = gradient;
    cut(k);
    return by_type(a->type, [&](auto t) {
        typedef decltype(t) T;
        return short_row<T>(k) ? run_gradient<T, 64>(k, (hipStream_t)stream) : run_gradient<T, 256>(k, (hipStream_t)stream);
    });
}

}  // extern "C"
