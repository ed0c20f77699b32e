// token_logprobs.hip -- log-probabilities of given tokens, with entropy and the most likely alternatives, and their gradient.
//
//   with the largest m:  log S = log sum_j exp(l_j - m),  logprob = (l_tok - m) - log S,  p_j = exp((l_j - m) - log S),
//   entropy = log S - sum_j p_j (l_j - m);    d(w logprob + u entropy) / d l_j = w ([j = tok] - p_j) - u p_j (log p_j + entropy)
//
// Differences from the largest, nowhere of large numbers.  A workgroup takes a row and reads it once: a thread holds a
// reference that is at most kSlack below its largest logit so far, sum e and sum d e with d = l - reference, e = exp d; when
// a vector passes the reference by more, the sums follow it.  The threads' join in a fixed order.
//
// The alternatives: 256 strips of the row (a thread's vectors, or four neighbours') each know their largest logit and the vector
// where it came first.  The k-th of these in the order of falling logits, then rising index, bounds the k largest from below,
// and they all lie in the k strips that are not behind it: only those are read again, what is not below the bound goes to a
// list, and the list is ranked entry against entry.  Where the list would overflow (strips whose logits lie high together) the
// row is passed over k times for the next largest instead.
//
// Where the weights of the gradient are known the row is read again at once, from the caches, and the gradient written.
// Bound by bytes for many rows; of one row by the vector instructions of its one CU, about 11 a logit.
#include <algorithm>

#include "rows.hpp"

namespace clear {
namespace {

constexpr uint32_t kMostTop = 32, kStrips = 256, kList = 1024;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f;
constexpr float kLowest = -3.40282347e38f, kSlack = 5.5f;
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
};

// what is known of a part of a row: its largest, and with e = exp(l - m): sum e, sum (m - l) e
struct Part {
    float m, s, t;
};
__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ inline Part joined(Part a, Part b) {
    const float m = a.m > b.m ? a.m : b.m;
    const float da = a.m == m ? 0.f : m - a.m, db = b.m == m ? 0.f : m - b.m;  // none where both are -inf
    const float ea = exp_of(-da), sa = a.s * ea, eb = exp_of(-db), sb = b.s * eb;
    return {m, sa + sb, (a.t * ea + (sa > 0.f ? da * sa : 0.f)) + (b.t * eb + (sb > 0.f ? db * sb : 0.f))};
}

template <int kThreads>
struct Shared {
    Part part[kThreads / 64];
    uint64_t best[kStrips], list[kList];
    uint32_t chosen[kMostTop];
    uint64_t bound;
    uint32_t listed, strips;
    uint64_t wave[kThreads / 64];
};

template <int kControl>
__device__ inline uint64_t swapped64(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, kControl, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), kControl, 0xf, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}

// An entry's place in the order: its logit's key, then the flipped index; 0 for what is no alternative.
__device__ inline uint64_t entry(float x, uint32_t index) {
    const uint32_t k = key_of(x);
    return k ? (uint64_t)k << 32 | (uint32_t)~index : 0;
}

// The k largest entries below `under` are found one by one where the list does not hold them.
template <class T, int kThreads>
__device__ void one_by_one(const Row<T, kThreads>& row, uint32_t k, Shared<kThreads>& s) {
    uint64_t under = ~0ull;
    for (uint32_t i = 0; i < k; i++) {
        uint64_t best = 0;
        for (int j = 0; j < row.vectors; j++) {
            float f[Row<T, kThreads>::V];
            const int v = j * kThreads + threadIdx.x;
            row.read(v, f);
#pragma unroll
            for (int c = 0; c < Row<T, kThreads>::V; c++) {
                const uint64_t e = entry(f[c], v * Row<T, kThreads>::V + c - row.skip);
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
    __syncthreads();
}

// The row's k largest to a.top, from each thread's largest `m` and the vector `first` where it came first.
template <class T, int kThreads>
__device__ void alternatives(const Args& a, const Row<T, kThreads>& row, uint32_t r, float mine, int first, float m, float logs,
                             Shared<kThreads>& s) {
    constexpr int V = Row<T, kThreads>::V, kEach = kThreads / kStrips;  // threads of a strip
    // ordered by a vector's first index; the bound takes its last, as the logit itself may lie anywhere in it
    uint64_t best = entry(mine, (uint32_t)(first * kThreads + (int)threadIdx.x) * V);
    if constexpr (kEach == 4) {
        uint64_t other = swapped64<0xb1>(best);
        best = other > best ? other : best;
        other = swapped64<0x4e>(best);
        best = other > best ? other : best;
    }
    const uint32_t strip = threadIdx.x / kEach;
    if (threadIdx.x % kEach == 0) s.best[strip] = best;
    if (threadIdx.x == 0) s.listed = s.strips = 0, s.bound = 0;
    __syncthreads();
    uint32_t rank = 0;
    {
        constexpr int kPart = kStrips / kEach;  // each of a strip's threads compares it with a part of the others
        const uint32_t from = threadIdx.x % kEach * kPart;
#pragma unroll 8
        for (int i = 0; i < kPart; i++) rank += s.best[from + i] > best;
        if constexpr (kEach == 4) {
            rank += __builtin_amdgcn_update_dpp(0, (int)rank, 0xb1, 0xf, 0xf, false);
            rank += __builtin_amdgcn_update_dpp(0, (int)rank, 0x4e, 0xf, 0xf, false);
        }
    }
    if (best && rank < a.k && threadIdx.x % kEach == 0) {
        s.chosen[atomicAdd(&s.strips, 1u)] = strip;  // their order says nothing
        if (rank == a.k - 1) s.bound = best - (V - 1);
    }
    __syncthreads();
    const uint64_t bound = s.bound;
    const uint32_t per = (uint32_t)row.vectors * kEach, items = s.strips * per;
    for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
        const uint32_t q = i / per, j = i - q * per;
        const int v = (int)(j / kEach) * kThreads + (int)(s.chosen[q] * kEach + j % kEach);
        float f[V];
        row.read(v, f);
#pragma unroll
        for (int c = 0; c < V; c++) {
            const int at = v * V + c;  // bounds and entries by places that count from the vectors' beginning
            const uint64_t e = entry(f[c], at);
            if (e && e >= bound) {
                const uint32_t to = atomicAdd(&s.listed, 1u);
                if (to < kList) s.list[to] = e + row.skip;  // the flipped index of at - skip
            }
        }
    }
    __syncthreads();
    if (s.listed > kList) one_by_one(row, a.k, s);
    const uint32_t n = s.listed;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t x = s.list[i];
        uint32_t before = 0;
        for (uint32_t j = 0; j < n; j++) before += s.list[j] > x;
        if (before < a.k && x) {
            a.top[(size_t)r * a.k + before] = (uint32_t)~(uint32_t)x;
            a.top_logprobs[(size_t)r * a.k + before] = (of_key((uint32_t)(x >> 32)) - m) - logs;
        }
    }
    // fewer than k logits are numbers above -inf
    __syncthreads();
    uint32_t have = n;
    if (n && n <= a.k) {
        have = 0;
        for (uint32_t j = 0; j < n; j++) have += s.list[j] != 0;
    }
    for (uint32_t i = have + threadIdx.x; i < a.k; i += kThreads) {
        a.top[(size_t)r * a.k + i] = -1;
        a.top_logprobs[(size_t)r * a.k + i] = -INFINITY;
    }
    __syncthreads();
}

template <class T, int kThreads>
__device__ void write_gradient(const Args& a, uint32_t r, int64_t token, float m, float logs, float entropy) {
    const T* from = (const T*)a.logits + r * a.stride;
    T* to = (T*)a.grad + r * a.grad_stride;
    const Row<T, kThreads> row(from, a.vocab);
    constexpr int V = Row<T, kThreads>::V;
    const float w = token >= 0 && a.weights ? a.weights[r] : 0.f, u = a.entropy_weights ? a.entropy_weights[r] : 0.f;
    const bool nothing = (w == 0.f && u == 0.f) || (m == -INFINITY && logs == 0.f);  // whatever the logits are
    const bool same = ((uintptr_t)from ^ (uintptr_t)to) % 16 == 0;
    const int at_token = nothing || token < 0 ? -1 : (int)token + row.skip;
    to -= row.skip;
    for (int j = 0; j < row.vectors; j++) {
        const int v = j * kThreads + threadIdx.x, at = v * V;
        float f[V];
        if (at >= row.end) break;
        if (nothing) {
#pragma unroll
            for (int c = 0; c < V; c++) f[c] = 0.f;
        } else {
            row.read(v, f);
#pragma unroll
            for (int c = 0; c < V; c++) {
                const float log = (f[c] - m) - logs, p = exp_of(log);
                f[c] = p == 0.f ? 0.f : -p * (w + u * (log + entropy));  // a log of -inf times 0 is 0; a NaN stays
                if (at + c == at_token) f[c] += w;
            }
        }
        if (same && at >= row.skip && at + V <= row.end) store<V>(to + at, f);
        else
#pragma unroll
            for (int c = 0; c < V; c++)
                if (at + c >= row.skip && at + c < row.end) to[at + c] = from_f32<T>(f[c]);
    }
}

// the token's place, -1 for one that is none
__device__ inline int64_t token_of(const Args& a, uint32_t r) {
    const int64_t token = a.tokens ? a.tokens[r] : -1;
    return token < (int64_t)a.vocab ? token : -1;
}

// kTop: alternatives are asked for; kGrad: the gradient too
template <class T, int kThreads, bool kTop, bool kGrad>
__global__ __launch_bounds__(kThreads) void k_logprobs(Args a) {
    __shared__ Shared<kThreads> s;
    constexpr int V = 16 / sizeof(T);
    const uint32_t r = blockIdx.x;
    const T* logits = (const T*)a.logits + r * a.stride;
    const Row<T, kThreads> row(logits, a.vocab);
    float reference = kLowest, largest = -INFINITY, sum = 0.f, along = 0.f;
    int first = 0;
    for (int j = 0; j < row.vectors; j += kFlight) {
        float f[kFlight][V];
#pragma unroll
        for (int i = 0; i < kFlight; i++) row.read((j + i) * kThreads + threadIdx.x, f[i]);
#pragma unroll
        for (int i = 0; i < kFlight; i++) {
            float m = f[i][0];
#pragma unroll
            for (int c = 1; c < V; c++) m = __builtin_fmaxf(m, f[i][c]);
            if (m > largest) largest = m, first = j + i;
            if (m - reference > kSlack) {
                const float d = __builtin_fminf(m - reference, 1e6f), e = exp_of(-d);
                along = (along - d * sum) * e;
                sum *= e;
                reference = m;
            }
#pragma unroll
            for (int c = 0; c < V; c++) {
                const float d = f[i][c] - reference, e = exp_of(d);
                sum += e;
                along += e * __builtin_fmaxf(d, kLowest);  // -inf weighs nothing
            }
        }
    }
    Part p{largest, sum, -along};
    if (largest > -INFINITY) {
        const float d = largest - reference, e = exp_of(-d);
        p.t = (d * sum - along) * e;
        p.s = sum * e;
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const Part q{__shfl_xor(p.m, o), __shfl_xor(p.s, o), __shfl_xor(p.t, o)};
        p = threadIdx.x & o ? joined(q, p) : joined(p, q);
    }
    if (threadIdx.x % 64 == 0) s.part[threadIdx.x / 64] = p;
    __syncthreads();
    p = s.part[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; w++) p = joined(p, s.part[w]);
    const bool none = p.m == -INFINITY && p.s == 0.f;  // nothing above -inf
    const float logs = none ? 0.f : __builtin_amdgcn_logf(p.s) * kLn2, entropy = none ? 0.f : logs + p.t / p.s;
    const int64_t token = token_of(a, r);
    if (threadIdx.x == 0) {
        if (a.logprobs) a.logprobs[r] = token < 0 ? 0.f : none ? -INFINITY : (to_f32(logits[token]) - p.m) - logs;
        if (a.entropy) a.entropy[r] = entropy;
        if (a.stats) {
            a.stats[2 * (size_t)r] = p.m;
            a.stats[2 * (size_t)r + 1] = logs;
        }
    }
    if constexpr (kTop) alternatives(a, row, r, largest, first, p.m, logs, s);
    if constexpr (kGrad) {
        __syncthreads();  // the gradient may take the logits' place, and their readers are done
        write_gradient<T, kThreads>(a, r, token, p.m, logs, entropy);
    }
}

template <class T, int kThreads>
__global__ __launch_bounds__(kThreads) void k_gradient(Args a) {
    const uint32_t r = blockIdx.x;
    write_gradient<T, kThreads>(a, r, token_of(a, r), a.stats[2 * (size_t)r], a.stats[2 * (size_t)r + 1],
                                a.entropy ? a.entropy[r] : 0.f);
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
// few rows: every thread that a CU has for a row; many: more workgroups, whose ends overlap
bool wide(const fhe_ssm_token_logprobs& a) { return a.rows <= 256 && a.vocab > 4096; }

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_token_logprobs_workspace(const fhe_ssm_token_logprobs* a, size_t* bytes) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (!bytes) return fail(CKKS_EINVAL, "token log-probabilities: null argument");
    *bytes = 0;
    return CKKS_OK;
}

int fhe_ssm_token_logprobs_forward(const fhe_ssm_token_logprobs* a, const void* logits, const int64_t* tokens,
                                   float* logprobs, float* entropy, float* statistics, int64_t* top, float* top_logprobs,
                                   const float* weights, const float* entropy_weights, void* gradient, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    using namespace clear;
    (void)workspace, (void)workspace_bytes;
    if (int rc = check(a)) return rc;
    if (a->rows == 0) return CKKS_OK;
    if (!logits || (logprobs && !tokens) || (a->top && (!top || !top_logprobs)) || (weights && !tokens))
        return fail(CKKS_EINVAL, "token log-probabilities: null argument");
    if (gradient)
        if (int rc = check_gradient(a, logits, gradient)) return rc;
    Args k = args(*a, logits, tokens);
    k.logprobs = logprobs, k.entropy = entropy, k.stats = statistics, k.top = top, k.top_logprobs = top_logprobs;
    k.weights = weights, k.entropy_weights = entropy_weights, k.grad = gradient;
    return by_type(a->type, [&](auto t) {
        typedef decltype(t) T;
        const auto run = [&](auto n, auto with_top, auto with_grad) {
            constexpr int kThreads = decltype(n)::value;
            hipLaunchKernelGGL((k_logprobs<T, kThreads, decltype(with_top)::value, decltype(with_grad)::value>), dim3(k.rows),
                               dim3(kThreads), 0, (hipStream_t)stream, k);
            return launched("token log-probabilities");
        };
        const auto of = [&](auto n) {
            const std::true_type yes;
            const std::false_type no;
            return k.k ? k.grad ? run(n, yes, yes) : run(n, yes, no) : k.grad ? run(n, no, yes) : run(n, no, no);
        };
        return wide(*a) ? of(std::integral_constant<int, 1024>{}) : of(std::integral_constant<int, 256>{});
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
    return by_type(a->type, [&](auto t) {
        typedef decltype(t) T;
        if (wide(*a)) hipLaunchKernelGGL((k_gradient<T, 1024>), dim3(k.rows), dim3(1024), 0, (hipStream_t)stream, k);
        else hipLaunchKernelGGL((k_gradient<T, 256>), dim3(k.rows), dim3(256), 0, (hipStream_t)stream, k);
        return launched("token log-probabilities: gradient");
    });
}

}  // extern "C"
