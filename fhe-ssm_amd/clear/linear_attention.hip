// linear_attention.hip -- linear attention with a decay for each head.
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t          (S: dk x dv, float32)
#include <algorithm>

#include "clear.hpp"

namespace clear {
namespace {

constexpr int kCols = 64;        // state columns of a workgroup
constexpr int kWaves = 4;        // its waves share the state's rows
constexpr int kGroup = 16;       // tokens whose queries and keys wait in LDS
constexpr uint32_t kMostKeys = 128;  // dk
constexpr float kFloor = -1000.f;    // exp of it is 0, and sums of it stay finite

struct Args {
    const void *q, *k, *v;
    const float* g;
    const int32_t* lengths;
    const float* state_in;
    float* state_out;
    void* out;
    uint32_t tokens, heads, q_each, k_each, dk, dv, tiles;
    float scale;
    int64_t qs[3], ks[3], vs[3], gs[3], os[3];
};

__device__ inline float floored(float g) { return g < kFloor ? kFloor : g; }  // a NaN stays one

// Token by token, the state in registers.  A workgroup holds 64 columns of one head's state (columns never meet); its four
// waves and their lanes share the rows: a lane holds V columns of R rows.  o_t is the sum over rows: lanes of a wave by
// shuffles, waves through LDS, once for 16 tokens.
template <class T, int V, int R>
__global__ __launch_bounds__(kWaves * 64) void k_recurrent(Args a) {
    constexpr int kColLanes = kCols / V, kRowLanes = 64 / kColLanes, kStep = kWaves * kRowLanes, kRows = kStep * R;
    __shared__ float s_q[kGroup][kRows], s_k[kGroup][kRows], s_part[kGroup][kWaves][kCols];
    __shared__ float s_g[kGroup];
    const uint32_t tile = blockIdx.x % a.tiles, item = blockIdx.x / a.tiles, h = item % a.heads, lane = item / a.heads;
    const int wave = threadIdx.x / 64, l = threadIdx.x % 64, row0 = wave * kRowLanes + l / kColLanes;
    const uint32_t col = tile * kCols + (l % kColLanes) * V;
    const bool cols_in = col + V <= a.dv;  // V = 4 only where dv is a multiple of 4
    const T* q = (const T*)a.q + lane * a.qs[0] + (h / a.q_each) * a.qs[2];
    const T* k = (const T*)a.k + lane * a.ks[0] + (h / a.k_each) * a.ks[2];
    const T* v = (const T*)a.v + lane * a.vs[0] + h * a.vs[2];
    const float* g = a.g + lane * a.gs[0] + h * a.gs[2];
    T* out = (T*)a.out + lane * a.os[0] + h * a.os[2];
    const int len = a.lengths ? min(max(a.lengths[lane], 0), (int)a.tokens) : (int)a.tokens;
    const size_t at = (size_t)item * a.dk * a.dv + col;

    float S[R][V];
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int c = 0; c < V; c++) S[i][c] = 0.f;
    if (a.state_in && cols_in) {
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint32_t row = row0 + i * kStep;
            if (row < a.dk) {
                if constexpr (V == 4) {
                    const f32x4 x = *(const f32x4*)(a.state_in + at + (size_t)row * a.dv);
#pragma unroll
                    for (int c = 0; c < V; c++) S[i][c] = x[c];
                } else
                    S[i][0] = a.state_in[at + (size_t)row * a.dv];
            }
        }
    }
    for (int t0 = 0; t0 < len; t0 += kGroup) {
        const int n = min(kGroup, len - t0);
        for (int e = threadIdx.x; e < n * kRows; e += blockDim.x) {
            const int t = e / kRows, i = e % kRows;
            s_q[t][i] = (uint32_t)i < a.dk ? to_f32(q[(t0 + t) * a.qs[1] + i]) : 0.f;
            s_k[t][i] = (uint32_t)i < a.dk ? to_f32(k[(t0 + t) * a.ks[1] + i]) : 0.f;
        }
        if ((int)threadIdx.x < n) s_g[threadIdx.x] = expf(floored(g[(t0 + (int)threadIdx.x) * a.gs[1]]));
        __syncthreads();
        for (int t = 0; t < n; t++) {
            float x[V], o[V];
#pragma unroll
            for (int c = 0; c < V; c++) {
                x[c] = cols_in ? to_f32(v[(t0 + t) * a.vs[1] + col + c]) : 0.f;
                o[c] = 0.f;
            }
            const float d = s_g[t];
#pragma unroll
            for (int i = 0; i < R; i++) {
                const float kk = s_k[t][row0 + i * kStep], qq = s_q[t][row0 + i * kStep];
#pragma unroll
                for (int c = 0; c < V; c++) {
                    S[i][c] = fmaf(d, S[i][c], kk * x[c]);
                    o[c] = fmaf(qq, S[i][c], o[c]);
                }
            }
#pragma unroll
            for (int c = 0; c < V; c++) {
#pragma unroll
                for (int m = kColLanes; m < 64; m *= 2) o[c] += __shfl_xor(o[c], m);
                if (l < kColLanes) s_part[t][wave][l * V + c] = o[c];
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < n * kCols; e += blockDim.x) {
            const int t = e / kCols, c = e % kCols;
            float o = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; w++) o += s_part[t][w][c];
            if (tile * kCols + c < a.dv) out[(t0 + t) * a.os[1] + tile * kCols + c] = from_f32<T>(o * a.scale);
        }
    }
    for (int e = len * kCols + threadIdx.x; e < (int)a.tokens * kCols; e += blockDim.x) {
        const uint32_t c = tile * kCols + e % kCols;
        if (c < a.dv) out[(e / kCols) * a.os[1] + c] = from_f32<T>(0.f);
    }
    if (a.state_out && cols_in) {
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint32_t row = row0 + i * kStep;
            if (row < a.dk) {
                if constexpr (V == 4) {
                    const f32x4 x = {S[i][0], S[i][1], S[i][2], S[i][3]};
                    *(f32x4*)(a.state_out + at + (size_t)row * a.dv) = x;
                } else
                    a.state_out[at + (size_t)row * a.dv] = S[i][0];
            }
        }
    }
}

template <class T, int V>
void launch_recurrent(const Args& a, uint32_t grid, hipStream_t st) {
    constexpr int step = kWaves * 64 / (kCols / V);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(kWaves * 64), 0, st, a); };
    if (a.dk <= 32) go(k_recurrent<T, V, 32 / step>);
    else if (a.dk <= 64) go(k_recurrent<T, V, 64 / step>);
    else go(k_recurrent<T, V, 128 / step>);
}

// ------------------------------------------------------------------------------------------------ host
int check(const fhe_ssm_linear_attention* a) {
    if (!a) return fail(CKKS_EINVAL, "linear attention: null description");
    if (a->type > FHE_SSM_F16) return fail(CKKS_EINVAL, "linear attention: unknown type %u", a->type);
    if (a->dk < 1 || a->dk > kMostKeys) return fail(CKKS_EINVAL, "linear attention: dk %u is not in [1, %u]", a->dk, kMostKeys);
    if (a->dv < 1 || a->heads < 1) return fail(CKKS_EINVAL, "linear attention: dv and heads are at least 1");
    if (a->q_heads < 1 || a->k_heads < 1 || a->heads % a->q_heads || a->heads % a->k_heads)
        return fail(CKKS_EINVAL, "linear attention: %u heads cannot share %u query and %u key heads", a->heads, a->q_heads,
                    a->k_heads);
    const uint64_t tiles = (a->dv + kCols - 1) / kCols;
    if ((uint64_t)a->lanes * a->heads > 0x7fffffffull / tiles || a->tokens > 0x1000000u)
        return fail(CKKS_EINVAL, "linear attention: too many lanes, heads or tokens");
    return CKKS_OK;
}

Args arguments(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v, const float* g,
               const int32_t* lengths, const float* state_in, float* state_out, void* out) {
    Args r{q, k, v, g, lengths, state_in, state_out, out, a->tokens, a->heads, a->heads / a->q_heads, a->heads / a->k_heads,
           a->dk, a->dv, (a->dv + kCols - 1) / kCols, a->scale, {}, {}, {}, {}, {}};
    for (int i = 0; i < 3; i++) {
        r.qs[i] = a->q_stride[i];
        r.ks[i] = a->k_stride[i];
        r.vs[i] = a->v_stride[i];
        r.gs[i] = a->decay_stride[i];
        r.os[i] = a->out_stride[i];
    }
    return r;
}

template <class F>
int by_type(uint32_t type, F&& f) {
    if (type == FHE_SSM_F32) f(0.f);
    else if (type == FHE_SSM_BF16) f(bf16{});
    else f(f16{});
    return CKKS_OK;
}

int run(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v, const float* g,
        const int32_t* lengths, const float* state_in, float* state_out, void* out, void* stream) {
    if (a->lanes == 0) return CKKS_OK;
    if (a->tokens && (!q || !k || !v || !g || !out)) return fail(CKKS_EINVAL, "linear attention: null argument");
    const Args r = arguments(a, q, k, v, g, lengths, state_in, state_out, out);
    const uint32_t grid = a->lanes * a->heads * r.tiles;
    const bool wide = a->dv % 4 == 0 && aligned(state_in, 16) && aligned(state_out, 16);
    by_type(a->type, [&](auto t) {
        if (wide) launch_recurrent<decltype(t), 4>(r, grid, (hipStream_t)stream);
        else launch_recurrent<decltype(t), 1>(r, grid, (hipStream_t)stream);
    });
    return launched("linear attention");
}

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_linear_attention_workspace(const fhe_ssm_linear_attention* a, size_t* bytes) {
    if (int rc = clear::check(a)) return rc;
    if (!bytes) return clear::fail(CKKS_EINVAL, "linear attention: null argument");
    *bytes = 0;
    return CKKS_OK;
}

int fhe_ssm_linear_attention_prompt(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v,
                                    const float* log_decay, const int32_t* lengths, const float* state_in,
                                    float* state_out, void* out, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    if (int rc = clear::check(a)) return rc;
    return clear::run(a, q, k, v, log_decay, lengths, state_in, state_out, out, stream);
}

int fhe_ssm_linear_attention_step(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v,
                                  const float* log_decay, const float* state_in, float* state_out, void* out,
                                  void* stream) {
    if (int rc = clear::check(a)) return rc;
    if (a->tokens != 1) return clear::fail(CKKS_EINVAL, "linear attention: a step has one token, not %u", a->tokens);
    return clear::run(a, q, k, v, log_decay, nullptr, state_in, state_out, out, stream);
}

}  // extern "C"
