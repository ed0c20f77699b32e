// layer_norm.hip -- layer norm over the channels of rows, and its gradient.
//
//   h = (x - mean) rstd,  y = h w + b;      with t = dy w:  dx = rstd (t - mean(t) - h mean(t h)),  dw = sum dy h,  db = sum dy
//
// Both are bound by the bytes of x, y and dy, dx: a row is read once and stays in registers, where its mean and then the sum of
// its squared distances from that mean are taken (a difference of two large sums would lose a row that lies far from 0).  L
// lanes share a row: 16, a wave, or a workgroup, whichever holds its channels at 4 to 32 a lane.  They walk on to other rows with
// the weights still in registers, and in the backward pass with their channels' sums of dw and db, which a workgroup joins in
// LDS and writes as one part; a second kernel adds the parts.  No order depends on timing.  The next row is on its way while one is
// worked on.
//
// 32,768 rows of 768 in bf16 take 17.2 us forward (5.8 TB/s) and 28.0 backward (5.4 TB/s) with 4.8 for the 256 parts.  (Weights
// read element by element: 35 forward, as every wave read them for four rows; without the next row on its way 33.4 backward.)
#include <algorithm>

#include "rows.hpp"

namespace clear {
namespace {

constexpr uint32_t kMostChannels = 16384;

struct Args {
    const void *x, *dy, *w, *b;
    void* y;  // the output, backward dx
    float *mean, *rstd, *dw, *db, *parts;
    uint32_t rows, d;
    bool wide;  // weights are float32
    int64_t xs, dys, ys;
    float eps, n, each;  // d as a float, and its reciprocal
};

// A row's elements of this lane as they lie in memory: group j of V lies at (j L + lane) V; none of a group past the row's end.
template <class T, int L, int V, int E>
struct Raw {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec v[E / V];
    __device__ void read(const T* p, uint32_t lane, uint32_t d) {
#pragma unroll
        for (int j = 0; j < E / V; j++) {
            const uint32_t i = (j * L + lane) * V;
            if (i < d) v[j] = *(const vec*)(p + i);
        }
    }
    // with zeros past the row's end
    __device__ void to(float (&f)[E], uint32_t lane, uint32_t d) const {
#pragma unroll
        for (int e = 0; e < E; e++) f[e] = (e / V * L + lane) * V < d ? to_f32((T)v[e / V][e % V]) : 0.f;
    }
};
template <int L, int V, int E, class T>
__device__ inline void store_row(T* p, uint32_t lane, uint32_t d, const float (&f)[E]) {
#pragma unroll
    for (int j = 0; j < E / V; j++) {
        const uint32_t i = (j * L + lane) * V;
        if (i < d) store<V>(p + i, f + j * V);
    }
}
// the lane's weights, zeros past the row's end
template <class T, int L, int V, int E>
__device__ inline void weights(const void* w, bool wide, uint32_t lane, uint32_t d, float none, float (&f)[E]) {
#pragma unroll
    for (int j = 0; j < E / V; j++) {
        const uint32_t i = (j * L + lane) * V;
#pragma unroll
        for (int c = 0; c < V; c++) f[j * V + c] = i + c < d ? none : 0.f;
        if (!w || i >= d) continue;
        if (!wide) load<V>((const T*)w + i, f + j * V);
        else
#pragma unroll
            for (int c = 0; c < V; c += 4) load<V < 4 ? V : 4>((const float*)w + i + c, f + j * V + c);
    }
}

constexpr int threads(int L, int most) { return L > 64 ? L : most; }  // of a workgroup

template <class T, int L, int V, int E>
__global__ __launch_bounds__(threads(L, 256)) void k_forward(Args a) {
    constexpr int kSlots = threads(L, 256) / L;
    __shared__ Sums<L, 1> s;
    const uint32_t lane = threadIdx.x % L;
    const uint32_t step = gridDim.x * kSlots;
    uint32_t row = blockIdx.x * kSlots + threadIdx.x / L;
    Raw<T, L, V, E> next;
    if (row < a.rows) next.read((const T*)a.x + row * a.xs, lane, a.d);
    float w[E], b[E];
    weights<T, L, V>(a.w, a.wide, lane, a.d, 1.f, w);
    weights<T, L, V>(a.b, a.wide, lane, a.d, 0.f, b);
    for (; row < a.rows; row += step) {
        float f[E];
        next.to(f, lane, a.d);
        if (row + step < a.rows) next.read((const T*)a.x + (row + step) * a.xs, lane, a.d);
        float sum[1] = {0.f};
#pragma unroll
        for (int e = 0; e < E; e++) sum[0] += f[e];
        sum_over<L>(sum, s, 0);
        const float mean = sum[0] / a.n;  // divided, so that a row of equal channels is at 0 from it
        sum[0] = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            f[e] = (e / V * L + lane) * V + e % V < a.d ? f[e] - mean : 0.f;
            sum[0] += f[e] * f[e];
        }
        sum_over<L>(sum, s, 1);
        const float rstd = 1.f / __builtin_sqrtf(sum[0] * a.each + a.eps);
#pragma unroll
        for (int e = 0; e < E; e++) f[e] = f[e] * rstd * w[e] + b[e];
        store_row<L, V>((T*)a.y + row * a.ys, lane, a.d, f);
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// kParam: dw and db are asked for
template <class T, int L, int V, int E, bool kParam>
__global__ __launch_bounds__(threads(L, 512)) void k_backward(Args a) {
    constexpr int kSlots = threads(L, 512) / L;
    __shared__ Sums<L, 2> s;
    const uint32_t lane = threadIdx.x % L, slot = threadIdx.x / L;
    const uint32_t step = gridDim.x * kSlots;
    uint32_t row = blockIdx.x * kSlots + slot;
    Raw<T, L, V, E> next, next_dy;
    if (row < a.rows) {
        next.read((const T*)a.x + row * a.xs, lane, a.d);
        next_dy.read((const T*)a.dy + row * a.dys, lane, a.d);
    }
    float w[E], dw[E], db[E];
    weights<T, L, V>(a.w, a.wide, lane, a.d, 1.f, w);
#pragma unroll
    for (int e = 0; e < E; e++) dw[e] = db[e] = 0.f;
    int turn = 0;
    for (; row < a.rows; row += step) {
        float h[E], t[E];
        next.to(h, lane, a.d);
        next_dy.to(t, lane, a.d);
        if (row + step < a.rows) {
            next.read((const T*)a.x + (row + step) * a.xs, lane, a.d);
            next_dy.read((const T*)a.dy + (row + step) * a.dys, lane, a.d);
        }
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < E; e++) {
            h[e] = (e / V * L + lane) * V + e % V < a.d ? (h[e] - mean) * rstd : 0.f;
            if constexpr (kParam) {
                dw[e] += t[e] * h[e];
                db[e] += t[e];
            }
            t[e] *= w[e];
            sum[0] += t[e];
            sum[1] += t[e] * h[e];
        }
        sum_over<L>(sum, s, turn);
        turn ^= 1;
        const float flat = sum[0] * a.each, along = sum[1] * a.each;
#pragma unroll
        for (int e = 0; e < E; e++) h[e] = rstd * (t[e] - flat - h[e] * along);
        store_row<L, V>((T*)a.y + row * a.ys, lane, a.d, h);
    }
    if constexpr (kParam) {
        // the slots' sums, the upper half's to the lower half's
        if constexpr (kSlots > 1) {
            __shared__ float half[kSlots / 2][2][E * L];
#pragma unroll
            for (int n = kSlots / 2; n > 0; n /= 2) {
                __syncthreads();
                if (slot >= n && slot < 2 * n)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        half[slot - n][0][e * L + lane] = dw[e];
                        half[slot - n][1][e * L + lane] = db[e];
                    }
                __syncthreads();
                if (slot < n)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        dw[e] += half[slot][0][e * L + lane];
                        db[e] += half[slot][1][e * L + lane];
                    }
            }
        }
        if (slot == 0) {
            float* part = a.parts ? a.parts + (size_t)blockIdx.x * 2 * a.d : nullptr;  // none: the one workgroup's are all
            float *to_w = part ? part : a.dw, *to_b = part ? part + a.d : a.db;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const uint32_t i = (e / V * L + lane) * V + e % V;
                if (i < a.d && to_w) to_w[i] = dw[e];
                if (i < a.d && to_b) to_b[i] = db[e];
            }
        }
    }
}

// The parts' sums: kCols columns of dw and db a workgroup, whose kSlices slices of threads take every so many-th part.
constexpr uint32_t kCols = 32, kSlices = 1024 / kCols;
__global__ __launch_bounds__(1024) void k_columns(const float* __restrict__ parts, uint32_t n, uint32_t d, float* dw, float* db) {
    __shared__ float s[kSlices][kCols];
    const uint32_t c = threadIdx.x % kCols, col = blockIdx.x * kCols + c, slice = threadIdx.x / kCols;
    float sum = 0.f;
    if (col < 2 * d)
#pragma unroll 16
        for (uint32_t p = slice; p < n; p += kSlices) sum += parts[(size_t)p * 2 * d + col];
    s[slice][c] = sum;
    __syncthreads();
    if (slice == 0 && col < 2 * d) {
        sum = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < kSlices; i++) sum += s[i][c];
        float* to = col < d ? dw : db;
        if (to) to[col < d ? col : col - d] = sum;
    }
}

// Which lanes share a row: the fewest that hold its channels, with vectors of 16 bytes where every row lies on them.  Without
// vectors a wave takes up to 16 elements a lane: 2,999 float32 rows of 1,101 took 8.6 + 10.9 us by workgroups of 256 with 8 a lane,
// 11.4 + 64 by waves with 32, each with twice today's parts of dw.  32 float32 elements a lane do not fit the backward pass'
// registers: 30,000 rows of 2,048 take 80 + 234 us by waves, 82 + 141 by workgroups; in bf16 41 + 71 and 43 + 88.
template <class T, class F>
int choose(bool vectors, uint32_t d, F&& f) {
    constexpr int V = 16 / sizeof(T);
#define CLEAR_FITS(L, E, W) \
    if (d <= (L) * (E)) return f(std::integral_constant<int, L>{}, std::integral_constant<int, E>{}, std::integral_constant<int, W>{})
    if (vectors) {
        CLEAR_FITS(16, 8, V);
        CLEAR_FITS(64, 8, V);
        CLEAR_FITS(64, 16, V);
        if constexpr (V == 4) {
            CLEAR_FITS(256, 8, V);
        } else {
            CLEAR_FITS(64, 32, V);
        }
        CLEAR_FITS(256, 16, V);
        CLEAR_FITS(256, 32, V);
        CLEAR_FITS(1024, 16, V);
    }
    CLEAR_FITS(16, 4, 1);
    CLEAR_FITS(64, 4, 1);
    CLEAR_FITS(64, 16, 1);
    CLEAR_FITS(256, 8, 1);
    CLEAR_FITS(256, 16, 1);
    CLEAR_FITS(1024, 16, 1);
#undef CLEAR_FITS
    return fail(CKKS_EINVAL, "layer norm: %u channels", d);
}

// the backward pass' workgroups, as many as its parts: 8 waves a CU (16: 31 us instead of 28 for 32,768 rows of 768)
template <class T>
uint32_t parts_of(bool vectors, uint32_t rows, uint32_t d) {
    return choose<T>(vectors, d, [&](auto l, auto, auto) {
        constexpr int L = decltype(l)::value, kSlots = threads(L, 512) / L;
        return (int)std::min<uint64_t>(((uint64_t)rows + kSlots - 1) / kSlots, 256 * 512 / threads(L, 512));
    });
}
uint32_t most_parts(const fhe_ssm_layer_norm& a) {
    const auto of = [&](auto t) {
        typedef decltype(t) T;
        return std::max(parts_of<T>(true, a.rows, a.channels), parts_of<T>(false, a.rows, a.channels));
    };
    return by_type(a.type, of);
}

int check(const fhe_ssm_layer_norm* a) {
    if (!a) return fail(CKKS_EINVAL, "layer norm: null description");
    if (a->type > FHE_SSM_F16) return fail(CKKS_EINVAL, "layer norm: unknown type %u", a->type);
    if (a->weight_type != FHE_SSM_F32 && a->weight_type != a->type)
        return fail(CKKS_EINVAL, "layer norm: weights of type %u are neither float32 nor like the rows", a->weight_type);
    if (a->channels < 1 || a->channels > kMostChannels) return fail(CKKS_EINVAL, "layer norm: %u channels", a->channels);
    if (a->rows > 0x7fffffffu) return fail(CKKS_EINVAL, "layer norm: too many rows");
    if (a->rows > 1 && (a->x_stride < 0 || a->dy_stride < 0 || a->out_stride < (int64_t)a->channels))
        return fail(CKKS_EINVAL, "layer norm: output rows overlap, or a negative stride");
    if (!(a->eps >= 0.f)) return fail(CKKS_EINVAL, "layer norm: eps below 0");
    return CKKS_OK;
}

Args args(const fhe_ssm_layer_norm& a, const void* x, const void* weight, void* y) {
    Args k{};
    k.x = x, k.w = weight, k.y = y;
    k.rows = a.rows, k.d = a.channels, k.wide = a.weight_type == FHE_SSM_F32;
    k.xs = a.x_stride, k.dys = a.dy_stride, k.ys = a.out_stride;
    k.eps = a.eps, k.n = (float)a.channels, k.each = 1.f / k.n;
    return k;
}

bool on_vectors(const void* p, int64_t stride, size_t size) { return aligned(p, 16) && stride * size % 16 == 0; }

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_layer_norm_workspace(const fhe_ssm_layer_norm* a, size_t* bytes) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (!bytes) return fail(CKKS_EINVAL, "layer norm: null argument");
    const uint32_t n = most_parts(*a);
    *bytes = n > 1 ? (size_t)n * 2 * a->channels * sizeof(float) : 0;
    return CKKS_OK;
}

int fhe_ssm_layer_norm_forward(const fhe_ssm_layer_norm* a, const void* x, const void* weight, const void* bias, void* out,
                               float* mean, float* rstd, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->rows == 0) return CKKS_OK;
    if (!x || !out) return fail(CKKS_EINVAL, "layer norm: null argument");
    Args k = args(*a, x, weight, out);
    k.b = bias, k.mean = mean, k.rstd = rstd;
    const auto run = [&](auto t) {
        typedef decltype(t) T;
        const size_t size = sizeof(T);
        const auto on = [&](const void* p, int64_t stride) { return on_vectors(p, k.rows > 1 ? stride : 0, size); };
        const bool vectors = k.d * size % 16 == 0 && aligned(weight, 16) && aligned(bias, 16) && on(x, k.xs) && on(out, k.ys);
        return choose<T>(vectors, k.d, [&](auto l, auto e, auto v) {
            constexpr int L = decltype(l)::value, E = decltype(e)::value, V = decltype(v)::value;
            constexpr int kThreads = threads(L, 256), kSlots = kThreads / L;
            const uint32_t blocks = std::min<uint32_t>((k.rows + kSlots - 1) / kSlots, 256 * 2048 / kThreads);
            hipLaunchKernelGGL((k_forward<T, L, V, E>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, k);
            return launched("layer norm");
        });
    };
    return by_type(a->type, run);
}

int fhe_ssm_layer_norm_backward(const fhe_ssm_layer_norm* a, const void* dy, const void* x, const void* weight,
                                const float* mean, const float* rstd, void* dx, float* dweight, float* dbias, void* workspace,
                                size_t workspace_bytes, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return fail(CKKS_EINVAL, "layer norm: null argument");
    Args k = args(*a, x, weight, dx);
    k.dy = dy, k.mean = (float*)mean, k.rstd = (float*)rstd, k.dw = dweight, k.db = dbias;
    const bool param = dweight || dbias;
    size_t need;
    if (int rc = fhe_ssm_layer_norm_workspace(a, &need)) return rc;
    if (param && need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return fail(CKKS_EINVAL, "layer norm: the workspace must have %zu bytes and lie on 16", need);
    const hipStream_t st = (hipStream_t)stream;
    const auto run = [&](auto t) {
        typedef decltype(t) T;
        const size_t size = sizeof(T);
        const auto on = [&](const void* p, int64_t stride) { return on_vectors(p, k.rows > 1 ? stride : 0, size); };
        const bool vectors = k.d * size % 16 == 0 && aligned(weight, 16) && on(x, k.xs) && on(dy, k.dys) && on(dx, k.ys);
        const uint32_t blocks = parts_of<T>(vectors, k.rows, k.d);
        k.parts = blocks > 1 ? (float*)workspace : nullptr;
        if (blocks)
            if (int rc = choose<T>(vectors, k.d, [&](auto l, auto e, auto v) {
                    constexpr int L = decltype(l)::value, E = decltype(e)::value, V = decltype(v)::value;
                    const dim3 grid(blocks), block(threads(L, 512));
                    if (param) hipLaunchKernelGGL((k_backward<T, L, V, E, true>), grid, block, 0, st, k);
                    else hipLaunchKernelGGL((k_backward<T, L, V, E, false>), grid, block, 0, st, k);
                    return launched("layer norm: gradient");
                }))
                return rc;
        if (!param || blocks == 1) return (int)CKKS_OK;
        hipLaunchKernelGGL(k_columns, dim3((2 * k.d + kCols - 1) / kCols), dim3(1024), 0, st, k.parts, blocks, k.d, dweight, dbias);
        return launched("layer norm: the weight's gradient");
    };
    return by_type(a->type, run);
}

}  // extern "C"
