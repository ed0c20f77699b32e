// gated_recurrence.hip -- the gated linear recurrence over a prompt, its gradient, and its step of one token.
//
//   a_t = sigmoid(z_t),   h_t = a_t h_{t-1} + (1 - a_t) x_t                          (per channel; h in float32)
//   d_t = dy_t + c_t,   c_{t-1} = a_t d_t,   dx_t = (1 - a_t) d_t,   dz_t = a_t (1 - a_t) d_t (h_{t-1} - x_t)
//
// c after the last token is the gradient of the state that is handed on, c before the first that of the state it began with.
// A run of tokens maps h to A h + H and, backwards, c to A c + G, with the same A, the product of its a.
//
// A workgroup has 64 channels of a lane and goes over its tokens tile by tile: each of its eight waves loads 12 tokens, folds
// them to A and H (and G), and finds the state before its own tokens from those of the waves before it, through LDS with one
// barrier a tile.  So every input is read once, in rows of 64 channels, and no token waits for more than its own wave's.  The
// backward pass needs h again, which it forms from z and x as it reads them anyway, from the states at the tiles' beginnings
// that the forward pass kept (one float a channel for 96 tokens); so it reads no outputs, and h is float32 whatever their type.
// Few lanes with many tokens are cut into segments of tiles: a first pass folds every segment to one A and H (or G), and a
// segment's workgroup begins with those of the segments before it.  Then the inputs are read twice.
//
// Bound by bytes where lanes fill the GPU: 32 float32 prompts of 1,024 tokens of 768 channels take 62 us forward and 101 backward
// (4.9 TB/s), in bf16, where a row of 64 channels is 128 bytes, 36 and 66; of lengths from 512 on 32 and 58, as the longest lane
// decides.  One float32 prompt of 16,384 tokens takes 17.8 to fold 35 segments and 26 for the outputs, backward 17.8 and 45.
// Texts of up to 12 tokens are taken by one wave, of up to 36 by three: 203 float32 lanes of 768 channels take 5.4 and 6.9 us for 12
// tokens, 11 and 18 for 36, with eight waves 19 and 29.
// Eight waves of 12 tokens: of 16 tokens 43 and 80 for the ragged prompts at the time, of 8 36 and 59, sixteen waves of 12 39 and
// 109, of 8 40 and 73.  Two bf16 channels a lane and two runs a wave, with tiles of 64 to 192 tokens, take the same time within
// 8 %, both ways.  About 20 (backward 32) vector instructions an element, a third of the cycles.
#include <algorithm>
#include <type_traits>

#include "rows.hpp"

namespace clear {
namespace {

constexpr int kWaves = 8, kRun = 12;      // waves of a workgroup; tokens of a wave
constexpr int kTile = kWaves * kRun;      // tokens between kept states
constexpr int kShort = 3;                 // waves for up to three runs
constexpr uint32_t kEnough = 512;         // workgroups: two for each CU

struct Args {
    const void *z, *x, *dy;
    void *out, *dz, *dx;
    const int32_t* lengths;
    const float* in;     // forward the state before, backward the gradient of the state after; null: 0
    float* last;         // forward the state after, backward the gradient of the state before
    float* saved;        // [lane][tile][channel]: states before tiles
    float* folded;       // of segments: [lane][segment][2][channel], then copies of `in` [lane][channel]
    uint32_t lanes, tokens, channels, strips, tiles, segments, each;  // each: tiles of a segment
    int64_t zs[2], xs[2], dys[2], outs[2], dzs[2], dxs[2];
};

// sigmoid(z) and sigmoid(-z).  A gate near 1 is 1 less the other, so that of the many that are multiplied each is rounded and no
// more (a reciprocal is off to one side).  The small one is off by up to (|z| + 4) 2^-24 of itself, as the exponent z log2(e) is
// rounded before its power is taken; below 2^-126 it is 0.
__device__ inline void gates(float z, float& a, float& rest) {
    const float e = __builtin_amdgcn_exp2f(1.44269504f * z);
    rest = __builtin_amdgcn_rcpf(1.f + e);
    a = z < 0.f ? e * rest : 1.f - rest;
}

__device__ inline uint32_t length_of(const Args& a, uint32_t lane) {
    return a.lengths ? (uint32_t)min(max(a.lengths[lane], 0), (int)a.tokens) : a.tokens;
}

// An element of a row that all lanes share, by its place in bytes.  (The row's address is kept from being taken apart into a sum
// for each lane and each row, which costs a vector instruction every time.)
template <class T>
__device__ inline __attribute__((address_space(1))) T& in_row(T* row, uint32_t bytes) {
    uint64_t at = (uint64_t)row;
    asm("" : "+s"(at));
    return *(__attribute__((address_space(1))) T*)(at + bytes);
}
// A wave's rows from t0 on as their bits, each in a register of its own (two 16-bit ones in one would be waited for to be put
// there); past `end` the last row again (kAll: none is).  `at` is the channel, or for lanes past the last that one.
template <bool kAll, class T>
__device__ inline void fetch(const T* rows, int64_t stride, uint32_t t0, uint32_t end, uint32_t at, uint32_t (&to)[kRun]) {
    typedef std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t> bits;
    const T* row = rows + (int64_t)(kAll ? t0 : min(t0, end - 1)) * stride;
#pragma unroll
    for (int i = 0; i < kRun; i++) {
        to[i] = in_row((const bits*)row, at * (uint32_t)sizeof(T));
        row += kAll || t0 + i + 1 < end ? stride : 0;
    }
}
template <bool kAll, class T>
__device__ inline void put(T* rows, int64_t stride, uint32_t t0, uint32_t end, uint32_t at, const float (&from)[kRun]) {
    T* row = rows + (int64_t)t0 * stride;
#pragma unroll
    for (int i = 0; i < kRun; i++, row += stride)
        if (kAll || t0 + i < end) in_row(row, at * (uint32_t)sizeof(T)) = from_f32<T>(from[i]);
}
template <class T>
__device__ inline float of_bits(uint32_t x) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(x);
    else return to_f32(__builtin_bit_cast(T, (uint16_t)x));
}

// the state (or gradient) that a segment begins with: what came in, through the segments before it (after it)
template <bool kBack>
__device__ inline float begin(const Args& a, uint32_t lane, uint32_t segment, uint32_t c) {
    if (a.segments == 1) return a.in ? a.in[(size_t)lane * a.channels + c] : 0.f;
    float s = a.folded[((size_t)a.lanes * a.segments * 2 + lane) * a.channels + c];
    const float* f = a.folded + (size_t)lane * a.segments * 2 * a.channels + c;
    const uint32_t n = kBack ? a.segments - 1 - segment : segment;
#pragma unroll 8
    for (uint32_t i = 0; i < n; i++) {
        const float* at = f + (size_t)(kBack ? a.segments - 1 - i : i) * 2 * a.channels;
        s = at[0] * s + at[a.channels];
    }
    return s;
}

// What the two passes' workgroups have in common: which lane, segment and channels are theirs.
template <int W>
struct Place {
    uint32_t lane, segment, c, from, wave, l, length, tile0, tile1, whole;  // whole: the end of the tiles that have all tokens
    bool in;
    size_t at;
    __device__ Place(const Args& a) {
        // workgroups go to the eight XCDs in turn; here each XCD gets neighbours, which read the same rows of memory
        const uint32_t most = gridDim.x / 8 * 8, id = blockIdx.x < most ? blockIdx.x % 8 * (most / 8) + blockIdx.x / 8 : blockIdx.x;
        const uint32_t strip = id % a.strips;
        segment = id / a.strips % a.segments, lane = id / a.strips / a.segments;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x % 64, c = strip * 64 + l;
        in = c < a.channels;
        from = min(c, a.channels - 1);
        length = length_of(a, lane);
        tile0 = segment * a.each, tile1 = min(a.tiles, tile0 + a.each);
        whole = max(tile0, min(tile1, length / (W * kRun)));
        at = (size_t)lane * a.channels + from;
    }
};

// The forward pass; !kOut: only the segments' A and H.  Tiles that have all their tokens come first, the rows of each on their
// way while the one before is worked on; then one that has some, and those behind the lane's length, which are zeros.
template <class T, bool kOut, int W>
__global__ __launch_bounds__(W * 64) void k_forward(Args a) {
    constexpr uint32_t kTile = W * kRun;
    __shared__ float s_a[2][W][64], s_h[2][W][64];
    const Place<W> p(a);
    const T *z = (const T*)a.z + p.lane * a.zs[0], *x = (const T*)a.x + p.lane * a.xs[0];
    T* out = kOut ? (T*)a.out + p.lane * a.outs[0] : nullptr;
    uint32_t zr[kRun], xr[kRun];
    const auto next = [&](auto all, uint32_t tile) {
        fetch<all.value>(z, a.zs[1], tile * kTile + p.wave * kRun, p.length, p.from, zr);
        fetch<all.value>(x, a.xs[1], tile * kTile + p.wave * kRun, p.length, p.from, xr);
    };
    if (p.tile0 < p.whole) next(std::true_type{}, p.tile0);
    float state = kOut ? begin<false>(a, p.lane, p.segment, p.from) : 0.f, product = 1.f;
    const auto work = [&](auto all, uint32_t tile) {
        constexpr bool kAll = all.value;
        const uint32_t t0 = tile * kTile + p.wave * kRun;
        if (kOut && a.saved && p.wave == 0 && p.in) a.saved[((size_t)p.lane * a.tiles + tile) * a.channels + p.c] = state;
        float g[kRun], b[kRun], A = 1.f, H = 0.f;
#pragma unroll
        for (int i = 0; i < kRun; i++) {
            float rest;
            gates(of_bits<T>(zr[i]), g[i], rest);
            b[i] = rest * of_bits<T>(xr[i]);
            if (!kAll && t0 + i >= p.length) g[i] = 1.f, b[i] = 0.f;  // a token that is not there keeps the state
        }
        if (kAll && tile + 1 < p.whole) next(all, tile + 1);
#pragma unroll
        for (int i = 0; i < kRun; i++) {
            H = g[i] * H + b[i];
            A *= g[i];
        }
        const int turn = tile & 1;
        s_a[turn][p.wave][p.l] = A;
        s_h[turn][p.wave][p.l] = H;
        __syncthreads();
        float mine = state;
#pragma unroll
        for (uint32_t w = 0; w < W; w++) {
            if (w == p.wave) mine = state;
            state = s_a[turn][w][p.l] * state + s_h[turn][w][p.l];
            if (!kOut) product *= s_a[turn][w][p.l];
        }
        if (kOut) {
#pragma unroll
            for (int i = 0; i < kRun; i++) {
                b[i] = mine = g[i] * mine + b[i];
                if (!kAll && t0 + i >= p.length) b[i] = 0.f;
            }
            if (p.in) put<kAll>(out, a.outs[1], t0, a.tokens, p.c, b);
        }
    };
    for (uint32_t tile = p.tile0; tile < p.whole; tile++) work(std::true_type{}, tile);
    for (uint32_t tile = p.whole; tile < p.tile1; tile++) {
        if (tile * kTile < p.length) {
            next(std::false_type{}, tile);
            work(std::false_type{}, tile);
        } else if (kOut && p.in) {
            const float none[kRun] = {};
            put<false>(out, a.outs[1], tile * kTile + p.wave * kRun, a.tokens, p.c, none);
        }
    }
    if (p.wave != 0 || !p.in) return;
    if (kOut) {
        if (a.last && p.segment == a.segments - 1) a.last[p.at] = state;
    } else {
        float* f = a.folded + ((size_t)p.lane * a.segments + p.segment) * 2 * a.channels + p.c;
        f[0] = product;
        f[a.channels] = state;
        // `in` and `last` may be one buffer, and workgroups of the second pass read the one while one of them writes the other
        if (p.segment == 0) a.folded[((size_t)a.lanes * a.segments * 2) * a.channels + p.at] = a.in ? a.in[p.at] : 0.f;
    }
}

// The backward pass, from the last tile to the first; !kOut: only the segments' A and G.
template <class T, bool kOut, int W>
__global__ __launch_bounds__(W * 64) void k_backward(Args a) {
    constexpr uint32_t kTile = W * kRun;
    __shared__ float s_a[2][W][64], s_h[2][W][64], s_g[2][W][64];
    const Place<W> p(a);
    const T *z = (const T*)a.z + p.lane * a.zs[0], *x = (const T*)a.x + p.lane * a.xs[0];
    const T* dy = a.dy ? (const T*)a.dy + p.lane * a.dys[0] : nullptr;
    T *dz = (T*)a.dz + p.lane * a.dzs[0], *dx = (T*)a.dx + p.lane * a.dxs[0];
    uint32_t zr[kRun], xr[kRun], dr[kRun];
    float h_next = 0.f;
    const auto next = [&](auto all, uint32_t tile) {
        const uint32_t t0 = tile * kTile + p.wave * kRun;
        fetch<all.value>(z, a.zs[1], t0, p.length, p.from, zr);
        if (kOut) fetch<all.value>(x, a.xs[1], t0, p.length, p.from, xr);
        if (dy) fetch<all.value>(dy, a.dys[1], t0, p.length, p.from, dr);
        else
#pragma unroll
            for (int i = 0; i < kRun; i++) dr[i] = 0;
        if (kOut) h_next = a.saved[((size_t)p.lane * a.tiles + tile) * a.channels + p.from];
    };
    float carry = kOut ? begin<true>(a, p.lane, p.segment, p.from) : 0.f, product = 1.f;
    const auto work = [&](auto all, uint32_t tile) {
        constexpr bool kAll = all.value;
        const uint32_t t0 = tile * kTile + p.wave * kRun;
        float g[kRun], r[kRun], b[kRun], d[kRun], h = h_next;
#pragma unroll
        for (int i = 0; i < kRun; i++) {
            gates(of_bits<T>(zr[i]), g[i], r[i]);
            b[i] = kOut ? of_bits<T>(xr[i]) : 0.f;
            d[i] = of_bits<T>(dr[i]);
            if (!kAll && t0 + i >= p.length) g[i] = 1.f, r[i] = b[i] = d[i] = 0.f;
        }
        if (kAll && tile > p.tile0) next(all, tile - 1);
        float A = 1.f, H = 0.f, G = 0.f;
#pragma unroll
        for (int i = 0; i < kRun; i++) {
            A *= g[i];
            H = g[i] * H + r[i] * b[i];
        }
#pragma unroll
        for (int i = kRun; i-- > 0;) G = g[i] * (G + d[i]);
        const int turn = tile & 1;
        s_a[turn][p.wave][p.l] = A;
        if (kOut) s_h[turn][p.wave][p.l] = H;
        s_g[turn][p.wave][p.l] = G;
        __syncthreads();
        float mine = carry;
#pragma unroll
        for (int w = W; w-- > 0;) {
            if ((uint32_t)w == p.wave) mine = carry;
            carry = s_a[turn][w][p.l] * carry + s_g[turn][w][p.l];
            if (!kOut) product *= s_a[turn][w][p.l];
        }
        if (kOut) {
#pragma unroll
            for (uint32_t w = 0; w < W - 1; w++)
                if (w < p.wave) h = s_a[turn][w][p.l] * h + s_h[turn][w][p.l];
#pragma unroll
            for (int i = 0; i < kRun; i++) {  // b: what dz takes besides d
                const float after = g[i] * h + r[i] * b[i];
                b[i] = g[i] * r[i] * (h - b[i]);
                h = after;
            }
#pragma unroll
            for (int i = kRun; i-- > 0;) {
                const float now = d[i] + mine;
                mine = g[i] * now;
                b[i] *= now;
                r[i] *= now;
                if (!kAll && t0 + i >= p.length) b[i] = r[i] = 0.f;
            }
            if (p.in) {
                put<kAll>(dz, a.dzs[1], t0, a.tokens, p.c, b);
                put<kAll>(dx, a.dxs[1], t0, a.tokens, p.c, r);
            }
        }
    };
    for (uint32_t tile = p.tile1; tile-- > p.whole;) {
        if (tile * kTile < p.length) {
            next(std::false_type{}, tile);
            work(std::false_type{}, tile);
        } else if (kOut && p.in) {
            const float none[kRun] = {};
            put<false>(dz, a.dzs[1], tile * kTile + p.wave * kRun, a.tokens, p.c, none);
            put<false>(dx, a.dxs[1], tile * kTile + p.wave * kRun, a.tokens, p.c, none);
        }
    }
    if (p.tile0 < p.whole) next(std::true_type{}, p.whole - 1);
    for (uint32_t tile = p.whole; tile-- > p.tile0;) work(std::true_type{}, tile);
    if (p.wave != 0 || !p.in) return;
    if (kOut) {
        if (a.last && p.segment == 0) a.last[p.at] = carry;
    } else {
        float* f = a.folded + ((size_t)p.lane * a.segments + p.segment) * 2 * a.channels + p.c;
        f[0] = product;
        f[a.channels] = carry;
        if (p.segment == 0) a.folded[((size_t)a.lanes * a.segments * 2) * a.channels + p.at] = a.in ? a.in[p.at] : 0.f;
    }
}

// One token for every lane: an element a thread.  Bound by its launch.
template <class T>
__global__ __launch_bounds__(256) void k_step(Args a) {
    const uint32_t at = blockIdx.x * 256 + threadIdx.x;
    if (at >= a.lanes * a.channels) return;
    const uint32_t lane = at / a.channels, c = at - lane * a.channels;
    float gate, rest;
    gates(to_f32(((const T*)a.z)[lane * a.zs[0] + c]), gate, rest);
    const float h = gate * (a.in ? a.in[at] : 0.f) + rest * to_f32(((const T*)a.x)[lane * a.xs[0] + c]);
    ((T*)a.out)[lane * a.outs[0] + c] = from_f32<T>(h);
    if (a.last) a.last[at] = h;
}

int check(const fhe_ssm_gated_recurrence* a) {
    if (!a) return fail(CKKS_EINVAL, "gated recurrence: null description");
    if (a->type > FHE_SSM_F16) return fail(CKKS_EINVAL, "gated recurrence: unknown type %u", a->type);
    if (a->channels < 1) return fail(CKKS_EINVAL, "gated recurrence: no channels");
    // a launch has less than 2^32 threads
    if (a->tokens > 1u << 24 || a->channels > 1u << 24 || (uint64_t)a->lanes * ((a->channels + 63) / 64) >= 1ull << 23)
        return fail(CKKS_EINVAL, "gated recurrence: too many tokens, lanes or channels");
    return CKKS_OK;
}

// rows of an output must not meet, whether they follow lane by lane or token by token
bool apart(const int64_t* s, const fhe_ssm_gated_recurrence& a) {
    const int64_t c = a.channels, n = a.tokens, m = a.lanes;
    if (n <= 1) return m <= 1 || s[0] >= c;
    if (m <= 1) return s[1] >= c;
    return (s[1] >= c && s[0] >= (n - 1) * s[1] + c) || (s[0] >= c && s[1] >= (m - 1) * s[0] + c);
}

void lay_out(Args& k, const fhe_ssm_gated_recurrence& a) {
    k.lanes = a.lanes, k.tokens = a.tokens, k.channels = a.channels;
    k.strips = (a.channels + 63) / 64;
    k.tiles = (a.tokens + kTile - 1) / kTile;
    // segments where lanes and strips leave CUs without work; each of two tiles at least
    const uint64_t have = (uint64_t)std::max(1u, a.lanes) * k.strips;
    uint32_t want = have >= kEnough / 2 ? 1 : (uint32_t)(kEnough / have);
    want = std::max(1u, std::min(want, k.tiles / 2));
    k.each = std::max(1u, (k.tiles + want - 1) / want);
    k.segments = std::max(1u, (k.tiles + k.each - 1) / k.each);
    for (int i = 0; i < 2; i++) k.zs[i] = a.z_stride[i], k.xs[i] = a.x_stride[i], k.outs[i] = a.out_stride[i];
}

size_t folded_bytes(const Args& k) {
    return k.segments > 1 ? (size_t)k.lanes * k.channels * (2 * k.segments + 1) * sizeof(float) : 0;
}

int workspace_of(Args& k, void* workspace, size_t bytes) {
    const size_t need = folded_bytes(k);
    if (need && (!workspace || !aligned(workspace, 16) || bytes < need))
        return fail(CKKS_EINVAL, "gated recurrence: the workspace must have %zu bytes and lie on 16", need);
    k.folded = (float*)workspace;
    return CKKS_OK;
}

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_gated_recurrence_workspace(const fhe_ssm_gated_recurrence* a, size_t* workspace_bytes, size_t* saved_bytes) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    Args k{};
    lay_out(k, *a);
    if (workspace_bytes) *workspace_bytes = folded_bytes(k);
    if (saved_bytes) *saved_bytes = (size_t)k.lanes * k.tiles * k.channels * sizeof(float);
    return CKKS_OK;
}

int fhe_ssm_gated_recurrence_prompt(const fhe_ssm_gated_recurrence* a, const void* z, const void* x, const int32_t* lengths,
                                    const float* state_in, float* state_out, void* out, void* saved, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->lanes == 0) return CKKS_OK;
    if (a->tokens && (!z || !x || !out)) return fail(CKKS_EINVAL, "gated recurrence: null argument");
    if (!apart(a->out_stride, *a)) return fail(CKKS_EINVAL, "gated recurrence: output rows overlap");
    Args k{};
    lay_out(k, *a);
    if (int rc = workspace_of(k, workspace, workspace_bytes)) return rc;
    if (!aligned(saved, 4)) return fail(CKKS_EINVAL, "gated recurrence: what is saved must lie on 4 bytes");
    k.z = z, k.x = x, k.out = out, k.lengths = lengths, k.in = state_in, k.last = state_out, k.saved = (float*)saved;
    return by_type(a->type, [&](auto t) {
        typedef decltype(t) T;
        const dim3 grid(k.lanes * k.segments * k.strips), block(kWaves * 64);
        if (k.segments > 1) hipLaunchKernelGGL((k_forward<T, false, kWaves>), grid, block, 0, (hipStream_t)stream, k);
        if (k.tokens <= kRun) hipLaunchKernelGGL((k_forward<T, true, 1>), grid, dim3(64), 0, (hipStream_t)stream, k);
        else if (k.tokens <= kShort * kRun) hipLaunchKernelGGL((k_forward<T, true, kShort>), grid, dim3(kShort * 64), 0, (hipStream_t)stream, k);
        else hipLaunchKernelGGL((k_forward<T, true, kWaves>), grid, block, 0, (hipStream_t)stream, k);
        return launched("gated recurrence");
    });
}

int fhe_ssm_gated_recurrence_backward(const fhe_ssm_gated_recurrence* a, const void* z, const void* x, const int32_t* lengths,
                                      const void* saved, const void* dout, const float* dstate_out, void* dz, void* dx,
                                      float* dstate_in, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->lanes == 0) return CKKS_OK;
    if (a->tokens && (!z || !x || !saved || !dz || !dx)) return fail(CKKS_EINVAL, "gated recurrence: null argument");
    if (!apart(a->dz_stride, *a) || !apart(a->dx_stride, *a)) return fail(CKKS_EINVAL, "gated recurrence: output rows overlap");
    Args k{};
    lay_out(k, *a);
    if (int rc = workspace_of(k, workspace, workspace_bytes)) return rc;
    if (!aligned(saved, 4)) return fail(CKKS_EINVAL, "gated recurrence: what is saved must lie on 4 bytes");
    k.z = z, k.x = x, k.dy = dout, k.dz = dz, k.dx = dx, k.lengths = lengths, k.in = dstate_out, k.last = dstate_in, k.saved = (float*)saved;
    for (int i = 0; i < 2; i++) k.dys[i] = a->dout_stride[i], k.dzs[i] = a->dz_stride[i], k.dxs[i] = a->dx_stride[i];
    return by_type(a->type, [&](auto t) {
        typedef decltype(t) T;
        const dim3 grid(k.lanes * k.segments * k.strips), block(kWaves * 64);
        if (k.segments > 1) hipLaunchKernelGGL((k_backward<T, false, kWaves>), grid, block, 0, (hipStream_t)stream, k);
        if (k.tokens <= kRun) hipLaunchKernelGGL((k_backward<T, true, 1>), grid, dim3(64), 0, (hipStream_t)stream, k);
        else if (k.tokens <= kShort * kRun) hipLaunchKernelGGL((k_backward<T, true, kShort>), grid, dim3(kShort * 64), 0, (hipStream_t)stream, k);
        else hipLaunchKernelGGL((k_backward<T, true, kWaves>), grid, block, 0, (hipStream_t)stream, k);
        return launched("gated recurrence: gradient");
    });
}

int fhe_ssm_gated_recurrence_step(const fhe_ssm_gated_recurrence* a, const void* z, const void* x, const float* state_in,
                                  float* state_out, void* out, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->tokens != 1) return fail(CKKS_EINVAL, "gated recurrence: a step has one token, not %u", a->tokens);
    if (a->lanes == 0) return CKKS_OK;
    if (!z || !x || !out) return fail(CKKS_EINVAL, "gated recurrence: null argument");
    if (!apart(a->out_stride, *a)) return fail(CKKS_EINVAL, "gated recurrence: output rows overlap");
    Args k{};
    lay_out(k, *a);
    k.z = z, k.x = x, k.out = out, k.in = state_in, k.last = state_out;
    const dim3 grid((uint32_t)(((uint64_t)k.lanes * k.channels + 255) / 256));
    return by_type(a->type, [&](auto t) {
        hipLaunchKernelGGL(k_step<decltype(t)>, grid, dim3(256), 0, (hipStream_t)stream, k);
        return launched("gated recurrence: step");
    });
}

}  // extern "C"
