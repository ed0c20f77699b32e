// linear_attention.hip -- linear attention with a decay for each head.
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t          (S: dk x dv, float32)
#include <algorithm>
#include <type_traits>

#include "clear.hpp"

namespace clear {
namespace {

constexpr int kCols = 64;        // state columns of a workgroup
constexpr int kWaves = 4;        // its waves share the state's rows
constexpr int kByToken = 4;      // the most tokens that go token by token
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

__device__ inline float power(float x) { return __builtin_amdgcn_exp2f(x); }  // 2^x, 0 below 2^-126
__device__ inline float floored(float g) { return g < kFloor ? kFloor : g; }  // a NaN stays one

// Token by token, the state in registers.  A workgroup holds 64 columns of one head's state (columns never meet); its four
// waves and their lanes share the rows: a lane holds V columns of R rows.  o_t is the sum over rows: lanes of a wave by
// shuffles, waves through LDS.  For up to four tokens; it is bound by its launch and by reading and writing the state once:
// 32 lanes of 12 heads of 64, 6.3 MB read and written, take 5.1 us in the kernel, one lane 4.2.
template <class T, int V, int R>
__global__ __launch_bounds__(kWaves * 64) void k_recurrent(Args a) {
    constexpr int kColLanes = kCols / V, kRowLanes = 64 / kColLanes, kStep = kWaves * kRowLanes, kRows = kStep * R;
    __shared__ float s_q[kByToken][kRows], s_k[kByToken][kRows], s_part[kByToken][kWaves][kCols];
    __shared__ float s_g[kByToken];
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
    for (int e = threadIdx.x; e < len * kRows; e += blockDim.x) {
        const int t = e / kRows, i = e % kRows;
        s_q[t][i] = (uint32_t)i < a.dk ? to_f32(q[t * a.qs[1] + i]) : 0.f;
        s_k[t][i] = (uint32_t)i < a.dk ? to_f32(k[t * a.ks[1] + i]) : 0.f;
    }
    if ((int)threadIdx.x < len) s_g[threadIdx.x] = expf(floored(g[(int)threadIdx.x * a.gs[1]]));
    __syncthreads();
    for (int t = 0; t < len; t++) {
        float x[V], o[V];
#pragma unroll
        for (int c = 0; c < V; c++) {
            x[c] = cols_in ? to_f32(v[t * a.vs[1] + col + c]) : 0.f;
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
    for (int e = threadIdx.x; e < len * kCols; e += blockDim.x) {
        const int t = e / kCols, c = e % kCols;
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) o += s_part[t][w][c];
        if (tile * kCols + c < a.dv) out[t * a.os[1] + tile * kCols + c] = from_f32<T>(o * a.scale);
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

// ------------------------------------------------------------------------------------------------ by chunks
// Chunks of 64 tokens, on the matrix cores.  With G_i the sum of the chunk's log decays up to token i:
//     o_i = exp(G_i) q_i S + sum_{j <= i} exp(G_i - G_j) (q_i . k_j) v_j,   S' = exp(G_63) S + sum_j exp(G_63 - G_j) k_j v_j^T
// The sums of decays and their differences are taken in 64 bits (in units of log 2): in 32 bits a chunk of strong decays would
// lose what its neighbouring tokens have in common.  Matrix operands are bf16 pieces of a value, each the upper 8 bits of what
// the ones before it left: one piece is a bf16 input, two a float16 one, three a float32 one.
// What is held in float32, the state, the scores and the decayed keys, goes in as three pieces for every type: with two the
// outputs of states and scores that cancel would be off by more than the rounding of a 16-bit output.
constexpr int kChunk = 64;
// Padding of rows in LDS, in 16-bit words.  kPad: 16 rows' reads of 16 bytes meet no bank more often than they must; kPadT: so
// do 16 channels' writes of four tokens, four rows apart, and reads of 8 bytes.
constexpr int kPad = 8, kPadT = 4;

constexpr int kWhole = 3;  // pieces of a float32
template <class X>
constexpr int kPieces = std::is_same<X, float>::value ? kWhole : std::is_same<X, f16>::value ? 2 : 1;  // of an input
// of a key for the scores, products of inputs alone: 16-bit ones go in as they are
template <class X>
constexpr int kKeyPieces = std::is_same<X, float>::value ? kWhole : 1;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// four floats as N pieces of four bf16 each; the last piece is rounded
template <int N>
__device__ inline void split4(const float (&x)[4], u32x2 (&to)[N]) {
    float f[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int p = 0; p < N; p++) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (p + 1 < N) {
                const uint32_t a = __float_as_uint(f[2 * i]) & 0xffff0000u, b = __float_as_uint(f[2 * i + 1]) & 0xffff0000u;
                to[p][i] = a >> 16 | b;
                f[2 * i] -= __uint_as_float(a);
                f[2 * i + 1] -= __uint_as_float(b);
            } else {
                typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
                to[p][i] = __builtin_bit_cast(uint32_t, bf16x2{(bf16)f[2 * i], (bf16)f[2 * i + 1]});
            }
        }
    }
}

// Channels d .. d + 3 of a row of `count`.  What lies outside is read from somewhere inside, so that no load waits for a
// branch, and made zero when it is used (keep): the loads of a chunk are under way while the one before is worked on, and a
// use of any would wait for them.  wide: rows lie on four elements and count is a multiple of 4.
template <class X>
struct Four {
    typedef X x4 __attribute__((ext_vector_type(4)));
    typedef typename std::conditional<sizeof(X) == 4, u32x4, uint32_t __attribute__((ext_vector_type(2)))>::type words;
    words raw;
    template <bool wide>
    __device__ __forceinline__ void load(const X* row, int d, int count) {
        if constexpr (wide) raw = *(const words*)(row + (d < count ? d : 0));
        else {
            x4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = row[d + i < count ? d + i : 0];
            raw = __builtin_bit_cast(words, v);
        }
    }
    __device__ __forceinline__ void keep(bool row, int d, int count) {  // zeros outside
        constexpr int each = sizeof(words) / sizeof(uint32_t) == 4 ? 1 : 2;
#pragma unroll
        for (int i = 0; i < 4 / each; i++) {
            uint32_t mask = 0;
#pragma unroll
            for (int e = 0; e < each; e++) mask |= (row & (d + i * each + e < count)) ? (each == 1 ? ~0u : 0xffffu << (16 * e)) : 0u;
            raw[i] &= mask;
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return to_f32((X)__builtin_bit_cast(x4, raw)[i]); }
};

// a row's four channels as they are in memory, in pieces; in one: as they are
template <class X, int N>
__device__ __forceinline__ void pieces(const Four<X>& x, u32x2 (&to)[N]) {
    if constexpr (N == 1) to[0] = x.raw;
    else {
        const float f[4] = {x[0], x[1], x[2], x[3]};
        split4(f, to);
    }
}

// c += a b over the pieces of both, the smallest first.  Pieces are cut off, so the second is below 2^-7 and the third below
// 2^-15 of the value; what is left out, the product of two third ones, is below 2^-30 of a product.
template <int A, int B>
__device__ inline f32x4 mma(const bf16x8 (&a)[A], const bf16x8 (&b)[B], f32x4 c) {
#pragma unroll
    for (int s = A + B - 2 < 3 ? A + B - 2 : 3; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < A; i++)
            if (s - i >= 0 && s - i < B) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
    return c;
}

// the same of 16-bit inputs as they are: their products are exact
template <class X>
__device__ inline f32x4 mma_inputs(bf16x8 a, bf16x8 b, f32x4 c) {
    if constexpr (std::is_same<X, f16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ inline bf16x8 read8(const uint16_t* p) { return *(const bf16x8*)p; }
__device__ inline bf16x8 read44(const uint16_t* p, const uint16_t* q) {
    const u32x2 a = *(const u32x2*)p, b = *(const u32x2*)q;
    return __builtin_bit_cast(bf16x8, u32x4{a.x, a.y, b.x, b.y});
}

struct ChunkArgs {
    Args a;
    uint32_t segments, segment;  // a segment's tokens, a multiple of a chunk
    float* joint;                // [segment][lane, head][dk][dv]: what a segment adds to the state, then the state before it
    double* sums;                // [segment][lane, head]: the log decay of a segment
    bool wide_in, wide_out, near;  // near: a chunk's rows lie within 32-bit offsets
};

// What the outputs read, keys (a token a row) and the state before the chunk (a column a row), and what the state's update
// reads, decayed keys (a channel a row).  Of more than 64 channels the second takes the place of the first, at two barriers
// more, so that two workgroups fit a CU (4 prompts of 2,048, heads of 128: 141 against 102 us; of 64 it costs: 32 prompts of 512
// to 1024 85 against 89 us, in float16 101 against 108).  256 registers are then all that a lane has: the kernels that make
// outputs of heads above 64 spill 44 (bf16), 8 and 40 of them (32 columns, bf16 and float16).
template <class X, int DK, int TV>
struct KeysApart {
    uint16_t k[kKeyPieces<X>][kChunk][DK + kPad];
    uint16_t st[kWhole][TV][DK + kPad];
    uint16_t kt[kWhole][DK][kChunk + kPadT];
};
template <class X, int DK, int TV>
struct KeysInTurn {
    union {
        struct {
            uint16_t k[kKeyPieces<X>][kChunk][DK + kPad];
            uint16_t st[kWhole][TV][DK + kPad];
        };
        uint16_t kt[kWhole][DK][kChunk + kPadT];
    };
};
constexpr bool in_turn(int DK) { return DK > 64; }
template <class X, int DK, int TV>
struct ChunkShared : std::conditional<in_turn(DK), KeysInTurn<X, DK, TV>, KeysApart<X, DK, TV>>::type {
    uint16_t vt[kPieces<X>][TV][kChunk + kPadT];  // values, a channel a row
    double sum[kChunk];
    int poisoned;                                    // the last chunk (its first token + 1) with a value not finite
};

// A workgroup takes TV columns of one head's state over one segment of one lane's tokens.  Wave w has the outputs of tokens
// 16 w .. 16 w + 15 of a chunk (transposed: a lane has one token and four neighbouring channels) and a quarter of the state's
// 16 x 16 tiles.  The scores of a token, as they come out of one product (a lane: one query, four neighbouring keys), go into
// the next one without leaving their registers: the values are read in the order of keys that this makes.
// kOut: outputs from the state before the segment; otherwise what the segment adds to the state, and its log decay.
// It is bound by the latency of a chunk's chain (decays, LDS, scores, outputs, state; about 11,500 cycles of a wave, for 31 % of
// which it issues vector and for 10 % matrix instructions): 32 prompts of 512 to 1,024 tokens, 12 heads of 64, 120 MB, take 82
// to 87 us; one of 8,192 tokens 47 to 49 us, 14 of them for what segments add, 6.5 to join them and 28 for the outputs.
template <class X, int DK, int TV, bool kOut>
__global__ __launch_bounds__(256, (in_turn(DK) && sizeof(ChunkShared<X, DK, TV>) * 2 <= 160 << 10 ? 2 : 1)) void k_chunks(ChunkArgs c) {
    constexpr int P = kPieces<X>, PK = kKeyPieces<X>, KK = DK / 32, CT = TV / 16, ST = DK / 16 * CT / 4;
    constexpr int kKeyBlocks = DK * kChunk / 16 / 256 ? DK * kChunk / 16 / 256 : 1;  // 4 x 4 blocks of a thread
    constexpr int kValueBlocks = TV * kChunk / 16 / 256 ? TV * kChunk / 16 / 256 : 1;
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    auto& s = *(ChunkShared<X, DK, TV>*)shared_bytes;
    const Args& a = c.a;
    const uint32_t items = gridDim.x / c.segments / a.tiles;
    const uint32_t tile = blockIdx.x % a.tiles, item = blockIdx.x / a.tiles % items, seg = blockIdx.x / a.tiles / items;
    const uint32_t h = item % a.heads, lane = item / a.heads, col0 = tile * TV;
    const int wave = threadIdx.x / 64, l = threadIdx.x % 64, lr = l % 16, lg = l / 16;
    const X* q = (const X*)a.q + lane * a.qs[0] + (h / a.q_each) * a.qs[2];
    const X* k = (const X*)a.k + lane * a.ks[0] + (h / a.k_each) * a.ks[2];
    const X* v = (const X*)a.v + lane * a.vs[0] + h * a.vs[2] + col0;
    const float* g = a.g + lane * a.gs[0] + h * a.gs[2];
    X* out = (X*)a.out + lane * a.os[0] + h * a.os[2] + col0;
    const int len = a.lengths ? min(max(a.lengths[lane], 0), (int)a.tokens) : (int)a.tokens;
    const int first = (int)(seg * c.segment), last = min((int)min((uint64_t)(seg + 1) * c.segment, (uint64_t)a.tokens), len);
    const int dk = a.dk, cols = min((int)(a.dv - col0), TV);
    const size_t part = ((size_t)(kOut && c.segments == 1 ? 0 : seg) * items + item) * a.dk * a.dv;

    // a thread's 4 x 4 blocks (tokens by channels) of keys and values
    Four<X> kx[kKeyBlocks][4], vx[kValueBlocks][4], qx[KK][2];
    float gx = 0.f;
    // neighbouring lanes have neighbouring channels, whose loads come together
    const auto block = [&](int b, int width, int& token, int& channel) {
        const int at = threadIdx.x + 256 * b;
        channel = at % (width / 4) * 4;
        token = at / (width / 4) * 4;
    };
    const auto fetch_as = [&](int t0, auto how) __attribute__((always_inline)) {
        constexpr bool wide = decltype(how)::value;
        const int n = min(kChunk, last - t0);
        gx = g[(int64_t)(t0 + min(l, n - 1)) * a.gs[1]];
#pragma unroll
        for (int b = 0; b < kKeyBlocks; b++) {
            int t, d;
            block(b, DK, t, d);
#pragma unroll
            for (int i = 0; i < 4; i++) kx[b][i].template load<wide>(k + (int64_t)(t0 + min(t + i, n - 1)) * a.ks[1], d, dk);
        }
#pragma unroll
        for (int b = 0; b < kValueBlocks; b++) {
            int t, d;
            block(b, TV, t, d);
#pragma unroll
            for (int i = 0; i < 4; i++) vx[b][i].template load<wide>(v + (int64_t)(t0 + min(t + i, n - 1)) * a.vs[1], d, cols);
        }
        if constexpr (kOut) {
            const int t = wave * 16 + lr;
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    qx[kk][i].template load<wide>(q + (int64_t)(t0 + min(t, n - 1)) * a.qs[1], kk * 32 + lg * 8 + i * 4, dk);
        }
    };
    const auto cut = [&](int n) __attribute__((always_inline)) {  // of a chunk of n tokens: zeros past them and past the channels
        gx = l < n ? gx : 0.f;
#pragma unroll
        for (int b = 0; b < kKeyBlocks; b++) {
            int t, d;
            block(b, DK, t, d);
#pragma unroll
            for (int i = 0; i < 4; i++) kx[b][i].keep(t + i < n, d, dk);
        }
#pragma unroll
        for (int b = 0; b < kValueBlocks; b++) {
            int t, d;
            block(b, TV, t, d);
#pragma unroll
            for (int i = 0; i < 4; i++) vx[b][i].keep(t + i < n, d, cols);
        }
        if constexpr (kOut) {
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int i = 0; i < 2; i++) qx[kk][i].keep(wave * 16 + lr < n, kk * 32 + lg * 8 + i * 4, dk);
        }
    };
    // a whole chunk of whole rows: a uniform address for each load, and 32-bit offsets of the threads that stay
    uint32_t k_off[kKeyBlocks], v_off[kValueBlocks];
#pragma unroll
    for (int b = 0; b < kKeyBlocks; b++) {
        int t, d;
        block(b, DK, t, d);
        k_off[b] = ((uint32_t)t * (uint32_t)a.ks[1] + d) * sizeof(X);
    }
#pragma unroll
    for (int b = 0; b < kValueBlocks; b++) {
        int t, d;
        block(b, TV, t, d);
        v_off[b] = ((uint32_t)t * (uint32_t)a.vs[1] + d) * sizeof(X);
    }
    const uint32_t q_off = ((uint32_t)(wave * 16 + lr) * (uint32_t)a.qs[1] + lg * 8) * sizeof(X), g_off = (uint32_t)l * (uint32_t)a.gs[1] * 4;
    // in parts, between the steps of the chunk before: in one go they fill the queue of the memory unit, and the wave stands
    const auto fetch_whole = [&](int t0, int what) __attribute__((always_inline)) {
        typedef typename Four<X>::words words;
        if (what == 0) gx = *(const float*)((const char*)(g + (int64_t)t0 * a.gs[1]) + g_off);
#pragma unroll
        for (int b = 0; b < kKeyBlocks; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (what == 0) if (kKeyBlocks > 1 || DK == 64 || threadIdx.x < DK * kChunk / 16)
                    kx[b][i].raw = *(const words*)((const char*)(k + (int64_t)(t0 + i) * a.ks[1]) + k_off[b]);
#pragma unroll
        for (int b = 0; b < kValueBlocks; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (what == 1) if (kValueBlocks > 1 || TV == 64 || threadIdx.x < TV * kChunk / 16)
                    vx[b][i].raw = *(const words*)((const char*)(v + (int64_t)(t0 + i) * a.vs[1]) + v_off[b]);
        if (kOut && what == 2) {
            const char* row = (const char*)(q + (int64_t)t0 * a.qs[1]);
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int i = 0; i < 2; i++) qx[kk][i].raw = *(const words*)(row + q_off + (kk * 32 + i * 4) * (int)sizeof(X));
        }
    };
    const auto whole_rows = [&](int t0) { return c.near && dk == DK && cols == TV && last - t0 >= kChunk; };
    const auto fetch_cut = [&](int t0) __attribute__((always_inline)) {  // one branch for all loads: each of its own waited
        if (c.wide_in) fetch_as(t0, std::true_type{});
        else fetch_as(t0, std::false_type{});
    };

    // the state: tile i of this wave covers rows d0(i) .. + 15 and columns c0(i) .. + 15, a lane has column lr, rows 4 lg ..
    f32x4 S[ST];
    const auto d0 = [&](int i) { return (wave * ST + i) / CT * 16; };
    const auto c0 = [&](int i) { return (wave * ST + i) % CT * 16; };
    const float* from = kOut ? (c.segments == 1 ? a.state_in : c.joint) : nullptr;
#pragma unroll
    for (int i = 0; i < ST; i++) {
        S[i] = f32x4{0, 0, 0, 0};
        if (from && c0(i) + lr < cols) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int d = d0(i) + lg * 4 + r;
                if (d < dk) S[i][r] = from[part + (size_t)d * a.dv + col0 + c0(i) + lr];
            }
        }
    }
    if (threadIdx.x == 0) s.poisoned = 0;
    double total = 0.;
    if (first < last) fetch_cut(first);
    for (int t0 = first; t0 < last; t0 += kChunk) {
        // sums of the decays: lane l of every wave has token l
        if (last - t0 < kChunk || dk < DK || cols < TV) cut(last - t0);
        const double sum = wave_scan((double)floored(gx) * 1.4426950408889634), whole = from_lane(sum, 63);
        total += whole;
        const float weight = power((float)(whole - sum)), all = power((float)whole);
        __syncthreads();  // the chunk before has been read
        if (threadIdx.x < kChunk) s.sum[l] = sum;
        if constexpr (kOut) {
#pragma unroll
            for (int b = 0; b < kKeyBlocks; b++) {
                int t, d;
                block(b, DK, t, d);
                if (t < kChunk) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        u32x2 piece[PK];
                        pieces(kx[b][i], piece);
#pragma unroll
                        for (int p = 0; p < PK; p++) *(u32x2*)&s.k[p][t + i][d] = piece[p];
                    }
                }
            }
        }
        const auto decayed_keys = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < kKeyBlocks; b++) {
                int t, d;
                block(b, DK, t, d);
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = __shfl(weight, (t + i) % kChunk);
                if (t < kChunk) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float f[4] = {kx[b][0][e] * w[0], kx[b][1][e] * w[1], kx[b][2][e] * w[2], kx[b][3][e] * w[3]};
                        u32x2 piece[kWhole];
                        split4(f, piece);
#pragma unroll
                        for (int p = 0; p < kWhole; p++) *(u32x2*)&s.kt[p][d + e][t] = piece[p];
                    }
                }
            }
        };
        constexpr bool kLater = kOut && in_turn(DK);
        if constexpr (!kLater) decayed_keys();
        bool odd = false;
#pragma unroll
        for (int b = 0; b < kValueBlocks; b++) {
            int t, d;
            block(b, TV, t, d);
            if (t < kChunk) {
                if constexpr (P == 1) {  // the 16-bit values themselves, four tokens of a channel together
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t take = e % 2 ? 0x07060302u : 0x05040100u;
                        u32x2 turned;
                        turned.x = __builtin_amdgcn_perm(vx[b][1].raw[e / 2], vx[b][0].raw[e / 2], take);
                        turned.y = __builtin_amdgcn_perm(vx[b][3].raw[e / 2], vx[b][2].raw[e / 2], take);
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            odd |= (turned[i] & 0x7f80u) == 0x7f80u || (turned[i] & 0x7f800000u) == 0x7f800000u;
                        *(u32x2*)&s.vt[0][d + e][t] = turned;
                    }
                } else
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float f[4] = {vx[b][0][e], vx[b][1][e], vx[b][2][e], vx[b][3][e]};
#pragma unroll
                    for (int i = 0; i < 4; i++) odd |= !(fabsf(f[i]) < INFINITY);
                    u32x2 piece[P];
                    split4(f, piece);
#pragma unroll
                    for (int p = 0; p < P; p++) *(u32x2*)&s.vt[p][d + e][t] = piece[p];
                }
            }
        }
        if (kOut && odd) s.poisoned = t0 + 1;
        bf16x8 Q[KK][P], q_scores[KK][PK];  // for the state, and for the scores
        if constexpr (kOut) {
#pragma unroll
            for (int i = 0; i < ST; i++) {
                const float f[4] = {S[i][0], S[i][1], S[i][2], S[i][3]};
                u32x2 piece[kWhole];
                split4(f, piece);
#pragma unroll
                for (int p = 0; p < kWhole; p++) *(u32x2*)&s.st[p][c0(i) + lr][d0(i) + lg * 4] = piece[p];
            }
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                u32x2 piece[2][P];
#pragma unroll
                for (int i = 0; i < 2; i++) pieces(qx[kk][i], piece[i]);
#pragma unroll
                for (int p = 0; p < P; p++)
                    Q[kk][p] = __builtin_bit_cast(bf16x8, u32x4{piece[0][p].x, piece[0][p].y, piece[1][p].x, piece[1][p].y});
                if constexpr (PK == 1)
                    q_scores[kk][0] = __builtin_bit_cast(bf16x8, u32x4{qx[kk][0].raw.x, qx[kk][0].raw.y, qx[kk][1].raw.x, qx[kk][1].raw.y});
                else
#pragma unroll
                    for (int p = 0; p < PK; p++) q_scores[kk][p] = Q[kk][p];
            }
        }
        __syncthreads();
        const int t1 = t0 + kChunk;
        const bool more = t1 < last && whole_rows(t1);
        if (!kLater) {
            if (more) fetch_whole(t1, 0);
            else if (t1 < last) fetch_cut(t1);
        }

        if constexpr (kOut) {
            const double mine = s.sum[wave * 16 + lr];
            f32x4 O[CT];
            const float before = power((float)mine);
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                O[ct] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    bf16x8 st[kWhole];
#pragma unroll
                    for (int p = 0; p < kWhole; p++) st[p] = read8(&s.st[p][ct * 16 + lr][kk * 32 + lg * 8]);
                    O[ct] = mma(st, Q[kk], O[ct]);
                }
                O[ct] *= before;
            }
            if (more) fetch_whole(t1, 1);
            const bool poisoned = s.poisoned == t0 + 1;
#pragma unroll
            for (int pair = 0; pair < 2; pair++) {
                if (pair * 2 > wave) break;
                u32x2 piece[2][kWhole];
                float p4[2][4];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int jt = pair * 2 + u;
#pragma unroll
                    for (int r = 0; r < 4; r++) p4[u][r] = 0.f;
                    if (jt <= wave) {
                        f32x4 score = {0, 0, 0, 0};
#pragma unroll
                        for (int kk = 0; kk < KK; kk++) {
                            bf16x8 kr[PK];
#pragma unroll
                            for (int p = 0; p < PK; p++) kr[p] = read8(&s.k[p][jt * 16 + lr][kk * 32 + lg * 8]);
                            if constexpr (PK == 1) score = mma_inputs<X>(kr[0], q_scores[kk][0], score);
                            else score = mma(kr, q_scores[kk], score);
                        }
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int j = jt * 16 + lg * 4 + r;
                            const float p = score[r] * power((float)(mine - s.sum[j]));
                            p4[u][r] = j <= wave * 16 + lr ? p : 0.f;
                        }
                    }
                    split4(p4[u], piece[u]);
                }
                if (!poisoned) {
                    bf16x8 pr[kWhole];
#pragma unroll
                    for (int p = 0; p < kWhole; p++)
                        pr[p] = __builtin_bit_cast(bf16x8, u32x4{piece[0][p].x, piece[0][p].y, piece[1][p].x, piece[1][p].y});
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        bf16x8 vr[P];
#pragma unroll
                        for (int p = 0; p < P; p++) {
                            const uint16_t* row = &s.vt[p][ct * 16 + lr][pair * 32 + lg * 4];
                            vr[p] = read44(row, row + 16);
                        }
                        O[ct] = mma(vr, pr, O[ct]);
                    }
                } else {
                    // a value here is infinite or NaN: a product with a score of 0 would carry it to tokens before its own,
                    // so the sums are taken over each token's own past, one by one
                    for (int ct = 0; ct < CT; ct++)
                        for (int e = 0; e < 16; e++) {
                            float o = 0.f;
                            for (int u = 0; u < 2; u++)
                                for (int r = 0; r < 4; r++) {
                                    const int j = (pair * 2 + u) * 16 + lg * 4 + r;
                                    if (j > wave * 16 + lr) continue;
                                    float x = 0.f;
                                    for (int p = P - 1; p >= 0; p--)
                                        x += __uint_as_float((uint32_t)s.vt[p][ct * 16 + e][j] << 16);
                                    o = fmaf(p4[u][r], x, o);
                                }
                            o += __shfl_xor(o, 16);
                            o += __shfl_xor(o, 32);
                            if (e / 4 == lg)
#pragma unroll
                                for (int i = 0; i < CT; i++)
#pragma unroll
                                    for (int r = 0; r < 4; r++)
                                        if (i == ct && r == e % 4) O[i][r] += o;
                        }
                }
            }
            const int t = t0 + wave * 16 + lr;
            if (t < last) {
                X* row = out + (int64_t)t * a.os[1];
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    const int e = ct * 16 + lg * 4;
                    typedef X x4 __attribute__((ext_vector_type(4)));
                    x4 o;
#pragma unroll
                    for (int r = 0; r < 4; r++) o[r] = from_f32<X>(O[ct][r] * a.scale);
                    if (c.wide_out && e + 4 <= cols) *(x4*)(row + e) = o;
                    else
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (e + r < cols) row[e + r] = o[r];
                }
            }
        }
        if constexpr (kLater) {
            __syncthreads();  // keys and state have been read
            decayed_keys();
        }
        if (more) {
            if (!kOut) fetch_whole(t1, 1);
            fetch_whole(t1, 2);
            if (kLater) fetch_whole(t1, 0);
        } else if (kLater && t1 < last)
            fetch_cut(t1);
        if (kLater) __syncthreads();
#pragma unroll
        for (int i = 0; i < ST; i++) {
            S[i] *= all;
#pragma unroll
            for (int kk = 0; kk < kChunk / 32; kk++) {
                bf16x8 kt[kWhole], vt[P];
#pragma unroll
                for (int p = 0; p < kWhole; p++) kt[p] = read44(&s.kt[p][d0(i) + lr][kk * 32 + lg * 8], &s.kt[p][d0(i) + lr][kk * 32 + lg * 8 + 4]);
#pragma unroll
                for (int p = 0; p < P; p++) vt[p] = read44(&s.vt[p][c0(i) + lr][kk * 32 + lg * 8], &s.vt[p][c0(i) + lr][kk * 32 + lg * 8 + 4]);
                S[i] = mma(kt, vt, S[i]);
            }
        }
    }
    if constexpr (kOut) {  // the rows past a lane's length, each with the segment it lies in
        const int end = (int)min((uint64_t)(seg + 1) * c.segment, (uint64_t)a.tokens), zero = max(last, first);
        for (int e = threadIdx.x; e < (end - zero) * TV; e += 256)
            if (e % TV < cols) out[(int64_t)(zero + e / TV) * a.os[1] + e % TV] = (X)0.f;
    }
    float* into = kOut ? (seg + 1 == c.segments ? a.state_out : nullptr) : c.joint;
    const size_t into_at = kOut ? (size_t)item * a.dk * a.dv : part;
    if (into) {
#pragma unroll
        for (int i = 0; i < ST; i++)
            if (c0(i) + lr < cols) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int d = d0(i) + lg * 4 + r;
                    if (d < dk) into[into_at + (size_t)d * a.dv + col0 + c0(i) + lr] = S[i][r];
                }
            }
    }
    if (!kOut && tile == 0 && threadIdx.x == 0) c.sums[(size_t)seg * items + item] = total;
}

// What each segment but the last adds becomes the state before it, along the segments; the last one's is stored behind them.
// 64 threads and one head a workgroup, so that the segments' decays are read once by each wave (12 heads, 32 segments,
// 6.3 MB read and written: 6.5 us, of it about 2.5 the launch).  kBatch: loads in flight, past the last segment the last again.
constexpr int kJoinThreads = 64;
template <uint32_t kBatch>
__global__ __launch_bounds__(kJoinThreads) void k_join(ChunkArgs c) {
    const uint32_t square = c.a.dk * c.a.dv, e = blockIdx.x * kJoinThreads + threadIdx.x, item = blockIdx.y, items = gridDim.y;
    if (e >= square) return;
    const size_t at = (size_t)item * square + e, each = (size_t)items * square;
    float S = c.a.state_in ? c.a.state_in[at] : 0.f;
    for (uint32_t s0 = 0; s0 < c.segments; s0 += kBatch) {
        float add[kBatch], decay[kBatch];
#pragma unroll
        for (uint32_t i = 0; i < kBatch; i++) {
            const uint32_t s = min(s0 + i, c.segments - 2);
            add[i] = c.joint[s * each + at];
            decay[i] = power((float)c.sums[(size_t)s * items + item]);
        }
#pragma unroll
        for (uint32_t i = 0; i < kBatch; i++)
            if (s0 + i < c.segments) {
                c.joint[(s0 + i) * each + at] = S;
                S = fmaf(decay[i], S, add[i]);
            }
    }
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
    // workgroups of 256 threads, all of a launch below 2^32
    const uint64_t tiles = ((uint64_t)a->dv + 31) / 32;  // the narrowest that a kernel takes
    if ((uint64_t)a->lanes * a->heads > 0xffffffull / tiles || a->tokens > 0x1000000u)
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
auto by_type(uint32_t type, F&& f) {
    if (type == FHE_SSM_F32) return f(0.f);
    if (type == FHE_SSM_BF16) return f(bf16{});
    return f(f16{});
}

// how a prompt is cut: by token (segments 0), or by chunks in so many segments
// By token 12 heads of 64 take 4.2 us for one token, 9.8 for 8 and 0.9 for each more, by chunks 7.2 us for up to 64.
struct Plan {
    uint32_t tile, segments, segment;
    size_t sums_at, bytes;
};

Plan plan(const fhe_ssm_linear_attention* a) {
    Plan p{};
    if (a->tokens <= (uint32_t)kByToken || !a->lanes) return p;
    const uint32_t items = a->lanes * a->heads, chunks = (a->tokens + kChunk - 1) / kChunk;
    // 64 columns of the state to a workgroup, or 32 where that leaves the GPU empty, though their keys and scores are worked
    // out twice (12 heads of one prompt: 64 tokens 8.8 against 7.7 us, 2,048 27.4 against 26.5; 8,192 49 against 58).  The
    // three pieces of float32 leave LDS for two workgroups of 32 columns on a CU (4 prompts of 2,048: 82 against 73 us).
    const uint64_t wide = (uint64_t)items * ((a->dv + 63) / 64);
    p.tile = a->type == FHE_SSM_F32 || (wide <= 192 && wide * chunks <= 384) ? 32 : 64;
    const uint32_t groups = items * ((a->dv + p.tile - 1) / p.tile);
    p.segments = 1;
    // the chunks of a prompt one after the other, or in segments on 512 workgroups, with two launches more (12 heads of one
    // prompt: 256 tokens 16.1 against 14.7 us, 8,192 485 against 49, on 1,024 workgroups 52; 32 ragged prompts, which are 384
    // workgroups in themselves, 86 against 111)
    if (groups < 256 && chunks >= 4) p.segments = std::min(chunks, 512 / groups);
    const uint32_t each = (chunks + p.segments - 1) / p.segments;
    p.segment = each * kChunk;
    p.segments = (chunks + each - 1) / each;
    if (p.segments > 1) {
        p.sums_at = ((size_t)p.segments * items * a->dk * a->dv * 4 + 255) / 256 * 256;
        p.bytes = p.sums_at + (size_t)p.segments * items * 8;
    }
    return p;
}

template <class X, int DK, int TV>
int launch_chunks(const ChunkArgs& c, uint32_t items, hipStream_t st) {
    const uint32_t bytes = sizeof(ChunkShared<X, DK, TV>);
    // LDS past 64 KB is asked for by name
    const auto go = [&](auto kernel, const ChunkArgs& c) -> int {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return fail(CKKS_EHIP, "linear attention: %s", hipGetErrorString(e));
        hipLaunchKernelGGL(kernel, dim3(items * c.a.tiles * c.segments), dim3(256), bytes, st, c);
        return CKKS_OK;
    };
    if (c.segments > 1) {
        ChunkArgs before = c;  // what the last segment adds, nothing reads
        before.segments--;
        if (int rc = go(k_chunks<X, DK, TV, false>, before)) return rc;
        const uint32_t square = c.a.dk * c.a.dv;
        hipLaunchKernelGGL(c.segments > 9 ? k_join<32> : k_join<8>, dim3((square + kJoinThreads - 1) / kJoinThreads, items),
                           dim3(kJoinThreads), 0, st, c);
    }
    return go(k_chunks<X, DK, TV, true>, c);
}

// Rows of out that certainly meet: neighbours along an axis, closer than a row is long.
bool rows_meet(const fhe_ssm_linear_attention* a) {
    const uint32_t count[3] = {a->lanes, a->tokens, a->heads};
    for (int i = 0; i < 3; i++) {
        const int64_t s = a->out_stride[i];
        if (count[i] > 1 && s < (int64_t)a->dv && s > -(int64_t)a->dv) return true;
    }
    return false;
}

int run(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v, const float* g,
        const int32_t* lengths, const float* state_in, float* state_out, void* out, void* workspace,
        size_t workspace_bytes, void* stream) {
    if (a->lanes == 0) return CKKS_OK;
    if (a->tokens && (!q || !k || !v || !g || !out)) return fail(CKKS_EINVAL, "linear attention: null argument");
    if (a->tokens && rows_meet(a)) return fail(CKKS_EINVAL, "linear attention: rows of out overlap");
    Args r = arguments(a, q, k, v, g, lengths, state_in, state_out, out);
    const hipStream_t st = (hipStream_t)stream;
    const Plan p = plan(a);
    if (!p.segments) {
        const bool wide = a->dv % 4 == 0 && aligned(state_in, 16) && aligned(state_out, 16);
        by_type(a->type, [&](auto t) {
            const uint32_t grid = a->lanes * a->heads * r.tiles;
            if (wide) launch_recurrent<decltype(t), 4>(r, grid, st);
            else launch_recurrent<decltype(t), 1>(r, grid, st);
        });
        return launched("linear attention");
    }
    if (p.bytes && (!workspace || workspace_bytes < p.bytes || !aligned(workspace, 8)))
        return fail(CKKS_EINVAL, "linear attention: a workspace of %zu bytes on 8 is needed", p.bytes);
    r.tiles = (a->dv + p.tile - 1) / p.tile;
    const size_t four = 4 * type_bytes(a->type);
    const auto wide = [&](const void* at, const int64_t* stride, uint32_t channels) {
        return aligned(at, four) && channels % 4 == 0 && stride[0] % 4 == 0 && stride[1] % 4 == 0 && stride[2] % 4 == 0;
    };
    ChunkArgs c{r, p.segments, p.segment, (float*)workspace, (double*)((char*)workspace + p.sums_at),
                      wide(q, r.qs, a->dk) && wide(k, r.ks, a->dk) && wide(v, r.vs, a->dv), wide(out, r.os, a->dv), false};
    const auto small = [&](const int64_t* stride) { return stride[1] >= 0 && stride[1] < (1 << 22); };
    c.near = c.wide_in && small(r.qs) && small(r.ks) && small(r.vs) && small(r.gs);
    const uint32_t items = a->lanes * a->heads;
    const int rc = by_type(a->type, [&](auto t) {
        typedef decltype(t) X;
        if constexpr (!std::is_same<X, float>::value)
            if (p.tile == 64)
                return a->dk <= 32 ? launch_chunks<X, 32, 64>(c, items, st)
                     : a->dk <= 64 ? launch_chunks<X, 64, 64>(c, items, st)
                                   : launch_chunks<X, 128, 64>(c, items, st);
        return a->dk <= 32 ? launch_chunks<X, 32, 32>(c, items, st)
             : a->dk <= 64 ? launch_chunks<X, 64, 32>(c, items, st)
                           : launch_chunks<X, 128, 32>(c, items, st);
    });
    return rc ? rc : launched("linear attention");
}

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_linear_attention_workspace(const fhe_ssm_linear_attention* a, size_t* bytes) {
    if (int rc = clear::check(a)) return rc;
    if (!bytes) return clear::fail(CKKS_EINVAL, "linear attention: null argument");
    *bytes = clear::plan(a).bytes;
    return CKKS_OK;
}

int fhe_ssm_linear_attention_prompt(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v,
                                    const float* log_decay, const int32_t* lengths, const float* state_in,
                                    float* state_out, void* out, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    if (int rc = clear::check(a)) return rc;
    return clear::run(a, q, k, v, log_decay, lengths, state_in, state_out, out, workspace, workspace_bytes, stream);
}

int fhe_ssm_linear_attention_step(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v,
                                  const float* log_decay, const float* state_in, float* state_out, void* out,
                                  void* stream) {
    if (int rc = clear::check(a)) return rc;
    if (a->tokens != 1) return clear::fail(CKKS_EINVAL, "linear attention: a step has one token, not %u", a->tokens);
    return clear::run(a, q, k, v, log_decay, nullptr, state_in, state_out, out, nullptr, 0, stream);
}

}  // extern "C"
