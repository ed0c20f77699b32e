// embedding.hip -- rows of a table by token with a scale, and the table's gradient.
//
//   out_t = s E[id_t],    dE[v] = s sum over t with id_t = v of dy_t
//
// The gradient adds a token's rows in an order that its tokens alone decide, whatever runs when: the positions are sorted by token
// (stable, so that equal tokens keep their order), and a wave takes each token's run.  A frequent token's run would keep one wave
// for long: where kPiece sorted positions that begin at a multiple of kPiece are of one token, a wave of their own has added them
// before, and the run's wave takes the sums; of a run of 64 and more four waves add a quarter each.  So a token's sum is the same
// in every call with the same tokens, but where its run begins among the sorted ones, which other tokens decide, may change its
// last bits.  Both read whole rows and are bound by their bytes.  Rows of the table that no token names
// are set to 0 by workgroups that run beside the sort's.
//
// 32,768 tokens, one in 16 the most frequent, of 768 channels in bf16 into a table of 65,536 rows in float32: 41 us of sorting
// beside 201 MB that are set to 0 (4.9 TB/s; its four kernels alone take 25), 9 for pieces, 27 for runs of 10,400 tokens.
// (Pieces of 32 rows: 11 and 31, of 8: 12 and 28; a wave alone for a long run 39.)  The lookup takes 16 to 20.
//
// The sort goes by two digits of half the token's bits.  A digit's pass counts its values in every workgroup's part, and then
// each workgroup adds up what lies before its own and moves its positions; a wave ranks 64 of them by comparing digits bit by
// bit through ballots.  Up to kSmall positions one workgroup does both passes in LDS, in one launch.
#include <algorithm>

#include "rows.hpp"

namespace clear {
namespace {

constexpr uint32_t kPiece = 16, kFew = 1024, kSmall = 8192;
constexpr uint32_t kTile = 2048, kMostParts = 256, kDigits = 1024;  // sorted at a time by a workgroup; workgroups; values of a digit
constexpr uint32_t kMostVocab = 1u << 18, kMostTokens = 1u << 25;

struct Args {
    const int64_t* tokens;
    const void* from;  // the table, or the gradient of the rows
    void* to;          // the rows, or the table's gradient
    uint32_t n, vocab, d;
    int64_t from_stride, to_stride;
    float scale;
    bool add;
    // of the gradient
    uint32_t bits[2], tiles, parts;  // of the digits; tiles of a part; parts
    uint32_t *ids[2], *at[2];        // the sorted tokens and positions: [1] after the first digit, [0] after the second
    uint32_t* counts;                // [part][digit]
    float* sums;                     // [piece][d]
    // the table's gradient is set to 0 by zero_blocks workgroups beside a kernel: a range of words of 16 bytes, and with the
    // first of them what lies before and behind whole words, in units of 2 bytes
    uint32_t zero_blocks, edges[2];
    u32x4* zero_at;
    size_t zero_from, zero_to;
    uint16_t* edge[2];
};

// a token outside the vocabulary: behind all others
__device__ inline uint32_t id_of(const Args& a, uint32_t i) {
    const int64_t t = a.tokens[i];
    return t >= 0 && t < (int64_t)a.vocab ? (uint32_t)t : a.vocab;
}

// ---------------------------------------------------------------- lookup
// A vector of V a thread, kEach times, over all rows; where that is more than a launch has threads for, again.
template <class F, class T, int V>
__global__ __launch_bounds__(256) void k_lookup(Args a) {
    constexpr int kEach = 4;
    const uint32_t vectors = (a.d + V - 1) / V;
    const uint64_t all = (uint64_t)a.n * vectors;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 * kEach + threadIdx.x; at < all; at += (uint64_t)gridDim.x * 256 * kEach) {
        float f[kEach][V];
        T* to[kEach];
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const uint64_t i = min(at + k * 256, all - 1);
            uint32_t row, c;
            if (all <= 0xffffffffull) row = (uint32_t)i / vectors, c = ((uint32_t)i - row * vectors) * V;
            else row = (uint32_t)(i / vectors), c = (uint32_t)(i - (uint64_t)row * vectors) * V;
            const int64_t token = a.tokens[row];
            const bool in = token >= 0 && token < (int64_t)a.vocab;
            load<V>((const F*)a.from + (in ? token : 0) * a.from_stride + c, f[k]);
            to[k] = (T*)a.to + row * a.to_stride + c;
#pragma unroll
            for (int e = 0; e < V; e++) f[k][e] = in ? f[k][e] * a.scale : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kEach; k++)
            if (at + k * 256 < all) store<V>(to[k], f[k]);
    }
}

// Rows of 256 vectors and more: a workgroup has kEach vectors a thread of one row, which costs no division for each of them.
// (5,619 bf16 rows of 4,091, single elements: 28 us, by k_lookup 45; of 4,096 both 19.)
template <class F, class T, int V>
__global__ __launch_bounds__(256) void k_lookup_long(Args a) {
    constexpr uint32_t kEach = 4;
    const uint32_t vectors = (a.d + V - 1) / V, parts = (vectors + 256 * kEach - 1) / (256 * kEach);
    const uint64_t all = (uint64_t)a.n * parts;
    for (uint64_t at = blockIdx.x; at < all; at += gridDim.x) {
        const uint32_t row = all <= 0xffffffffull ? (uint32_t)at / parts : (uint32_t)(at / parts), part = (uint32_t)(at - (uint64_t)row * parts);
        const int64_t token = a.tokens[row];
        const bool in = token >= 0 && token < (int64_t)a.vocab;
        const F* from = (const F*)a.from + (in ? token : 0) * a.from_stride;
        T* to = (T*)a.to + row * a.to_stride;
        const uint32_t first = part * 256 * kEach + threadIdx.x;
        float f[kEach][V];
#pragma unroll
        for (uint32_t k = 0; k < kEach; k++) load<V>(from + min(first + k * 256, vectors - 1) * V, f[k]);
#pragma unroll
        for (uint32_t k = 0; k < kEach; k++) {
            if (first + k * 256 >= vectors) continue;
#pragma unroll
            for (int e = 0; e < V; e++) f[k][e] = in ? f[k][e] * a.scale : 0.f;
            store<V>(to + (first + k * 256) * V, f[k]);
        }
    }
}

// ---------------------------------------------------------------- the sort
struct Sort {
    uint16_t ranks[16][kDigits];  // of each wave: how many of a digit it has; later where its next one goes, from the part's begin
    uint32_t base[kDigits], wave[16];
};

// lanes of the wave whose digit is this one's
__device__ inline uint64_t equals(uint32_t digit, uint32_t bits, bool in) {
    uint64_t same = __ballot(in);
    for (uint32_t b = 0; b < bits; b++) {
        const uint64_t set = __ballot(digit >> b & 1);
        same &= digit >> b & 1 ? set : ~set;
    }
    return same;
}

// Of 1,024 values, one a thread: the sum of those before it.  Ends with a barrier.
__device__ inline uint32_t before(uint32_t x, uint32_t* wave) {
    const uint32_t upto = (uint32_t)wave_scan<uint64_t>(x);
    if (threadIdx.x % 64 == 63) wave[threadIdx.x / 64] = upto;
    __syncthreads();
    uint32_t sum = upto - x;
    for (uint32_t w = 0; w < threadIdx.x / 64; w++) sum += wave[w];
    __syncthreads();
    return sum;
}

// what the wave's lanes wrote to LDS before is what they read after; nothing is waited for, a wave's LDS operations are in order
__device__ inline void in_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Ranks the digits of up to 64 kRounds positions of each wave, kRounds rounds of 64 in order: after it, position (wave, round,
// lane) with digit x goes to s.ranks[wave][x] + rank[round], in the order of the tile.  Ends with a barrier.
template <int kRounds>
__device__ inline void rank_tile(Sort& s, const uint32_t (&digit)[kRounds], const bool (&in)[kRounds], uint32_t bits,
                                 uint32_t (&rank)[kRounds]) {
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    for (uint32_t i = lane; i < kDigits / 2; i += 64) ((uint32_t*)s.ranks[wave])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        const uint64_t same = equals(digit[r], bits, in[r]);
        const uint32_t low = __popcll(same & ((1ull << lane) - 1));
        const uint32_t have = in[r] ? s.ranks[wave][digit[r]] : 0;
        rank[r] = have + low;
        in_order();
        if (in[r] && low == 0) s.ranks[wave][digit[r]] = (uint16_t)(have + __popcll(same));
        in_order();
    }
    __syncthreads();
    // a digit a thread: the waves' counts become what lies before each wave; the digit's total is returned in base
    uint32_t sum = 0;
    for (int w = 0; w < 16; w++) {
        const uint32_t have = s.ranks[w][threadIdx.x];
        s.ranks[w][threadIdx.x] = (uint16_t)sum;
        sum += have;
    }
    s.base[threadIdx.x] = sum;
    __syncthreads();
}

// sets a part of the table's gradient to 0
__device__ inline void zero(const Args& a, uint32_t block) {
    const u32x4 none = {0, 0, 0, 0};
    for (size_t i = a.zero_from + (size_t)block * 1024 + threadIdx.x; i < a.zero_to; i += (size_t)a.zero_blocks * 1024) a.zero_at[i] = none;
    if (block == 0 && a.zero_from == 0)
        for (int e = 0; e < 2; e++)
            if (threadIdx.x < a.edges[e]) a.edge[e][threadIdx.x] = 0;
}

__global__ __launch_bounds__(1024) void k_zero(Args a) { zero(a, blockIdx.x); }

// Up to 1,024 kRounds positions in one workgroup; the others set to 0.
template <int kRounds>
__global__ __launch_bounds__(1024) void k_sort_small(Args a) {
    __shared__ Sort s;
    __shared__ uint32_t keys[kSmall];
    if (blockIdx.x > 0) return zero(a, blockIdx.x - 1);
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const uint32_t each = (a.n + 1023) / 1024 * 64;  // of a wave
    uint32_t key[kRounds], digit[kRounds], rank[kRounds];
    bool in[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        const uint32_t i = wave * each + r * 64 + lane;
        in[r] = (uint32_t)r * 64 < each && i < a.n;
        key[r] = in[r] ? id_of(a, i) << 13 | i : 0;  // 19 and 13 bits
    }
    static_assert(kMostVocab <= (1u << 19) - 1 && kSmall == 1u << 13);
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
        const uint32_t shift = 13 + (pass ? a.bits[0] : 0), bits = a.bits[pass];
#pragma unroll
        for (int r = 0; r < kRounds; r++) digit[r] = key[r] >> shift & ((1u << bits) - 1);
        rank_tile<kRounds>(s, digit, in, bits, rank);
        const uint32_t begin = before(s.base[threadIdx.x], s.wave);
        s.base[threadIdx.x] = begin;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRounds; r++)
            if (in[r]) keys[s.base[digit[r]] + s.ranks[wave][digit[r]] + rank[r]] = key[r];
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRounds; r++) {
            const uint32_t i = wave * each + r * 64 + lane;
            if (in[r]) key[r] = keys[i];
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        const uint32_t i = wave * each + r * 64 + lane;
        if (in[r]) a.ids[0][i] = key[r] >> 13, a.at[0][i] = key[r] & (kSmall - 1);
    }
}

template <int kPass>
__device__ inline uint32_t sorted_id(const Args& a, uint32_t i) {
    return kPass == 0 ? id_of(a, i) : a.ids[1][i];
}
template <int kPass>
__device__ inline uint32_t digit_of(const Args& a, uint32_t id) {
    return (kPass ? id >> a.bits[0] : id) & ((1u << a.bits[kPass]) - 1);
}

// How many positions of a part have each value of the digit.
template <int kPass>
__global__ __launch_bounds__(1024) void k_count(Args a) {
    __shared__ uint32_t s[kDigits];
    if (blockIdx.x >= a.parts) return zero(a, blockIdx.x - a.parts);
    s[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t from = blockIdx.x * a.tiles * kTile, upto = min(a.n, from + a.tiles * kTile);
    for (uint32_t i = from + threadIdx.x; i < upto; i += 1024) atomicAdd(&s[digit_of<kPass>(a, sorted_id<kPass>(a, i))], 1u);
    __syncthreads();
    a.counts[blockIdx.x * kDigits + threadIdx.x] = s[threadIdx.x];
}

// Moves a part's positions to where its digits go.
template <int kPass>
__global__ __launch_bounds__(1024) void k_move(Args a) {
    __shared__ Sort s;
    __shared__ uint32_t next[kDigits];
    if (blockIdx.x >= a.parts) return zero(a, blockIdx.x - a.parts);
    uint32_t all = 0, mine = 0;
#pragma unroll 8
    for (uint32_t p = 0; p < a.parts; p++) {
        const uint32_t c = a.counts[p * kDigits + threadIdx.x];
        mine += p < blockIdx.x ? c : 0;
        all += c;
    }
    next[threadIdx.x] = before(all, s.wave) + mine;
    __syncthreads();
    constexpr int kRounds = kTile / 1024;
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const uint32_t from = blockIdx.x * a.tiles * kTile;
    for (uint32_t tile = 0; tile < a.tiles; tile++) {
        uint32_t id[kRounds], at[kRounds], digit[kRounds], rank[kRounds];
        bool in[kRounds];
#pragma unroll
        for (int r = 0; r < kRounds; r++) {
            const uint32_t i = from + tile * kTile + (wave * kRounds + r) * 64 + lane;
            in[r] = i < a.n;
            id[r] = in[r] ? sorted_id<kPass>(a, i) : 0;
            at[r] = kPass == 0 ? i : in[r] ? a.at[1][i] : 0;
            digit[r] = digit_of<kPass>(a, id[r]);
        }
        rank_tile<kRounds>(s, digit, in, a.bits[kPass], rank);
#pragma unroll
        for (int r = 0; r < kRounds; r++)
            if (in[r]) {
                const uint32_t to = next[digit[r]] + s.ranks[wave][digit[r]] + rank[r];
                a.ids[1 - kPass][to] = id[r];
                a.at[1 - kPass][to] = at[r];
            }
        __syncthreads();
        next[threadIdx.x] += s.base[threadIdx.x];
    }
}

// ---------------------------------------------------------------- the gradient
// Channels of a wave: groups of V, kGroups of them a lane, then the next 64 V kGroups.  Single elements take more groups, so that
// as much of a row is on its way: 5,619 bf16 rows of 4,091 take 27 us for pieces and 78 for runs, with two groups 60 and 181.
template <int V>
constexpr int groups() { return V == 1 ? 8 : 2; }
constexpr int kFewGroups = 2;  // of k_few, whose waves share a row

// Adds n rows to f, in order; row(j) is where row j begins.  Up to kFlight rows are on their way at once, at the end the last
// of them again for those that are not there: a row that is waited for alone takes as long as all.  A lane past the row's end
// reads its beginning.
template <int kRows, int V, int N, class F>
__device__ inline void add_batch(uint32_t j, uint32_t n, const uint32_t (&c)[N / V], float (&f)[N], F&& row) {
    float x[kRows][N];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const auto* at = row(min(j + i, n - 1));
#pragma unroll
        for (int g = 0; g < N / V; g++) load<V>(at + c[g], x[i] + g * V);
    }
#pragma unroll
    for (int i = 0; i < kRows; i++)
#pragma unroll
        for (int e = 0; e < N; e++) f[e] = j + i < n ? f[e] + x[i][e] : f[e];
}
template <int kFlight, int V, int N, class F>
__device__ inline void add_rows(uint32_t n, uint32_t c0, uint32_t d, float (&f)[N], F&& row) {
    static_assert(kFlight >= 2);
    uint32_t c[N / V];
#pragma unroll
    for (int g = 0; g < N / V; g++) {
        c[g] = c0 + (g * 64 + threadIdx.x % 64) * V;
        c[g] = c[g] < d ? c[g] : 0;
    }
    for (uint32_t j = 0; j < n; j += kFlight) {
        if (n - j <= 2) add_batch<2, V>(j, n, c, f, row);
        else add_batch<kFlight, V>(j, n, c, f, row);
    }
}
// rows at .. at + n - 1 of 64 sorted positions, of which each lane holds one
template <class T, int kFlight, int V, int N>
__device__ inline void add_held(const Args& a, uint32_t held, uint32_t at, uint32_t n, uint32_t c0, float (&f)[N]) {
    add_rows<kFlight, V>(n, c0, a.d, f, [&](uint32_t j) {
        return (const T*)a.from + (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)held, (int)(at + j)) * a.from_stride;
    });
}

// scales a row's sum and writes it, or adds it to what is there
template <class G, int V, int N>
__device__ inline void write_row(const Args& a, uint32_t id, uint32_t c0, float (&f)[N]) {
    G* to = (G*)a.to + (size_t)id * a.d;
#pragma unroll
    for (int g = 0; g < N / V; g++) {
        const uint32_t c = c0 + (g * 64 + threadIdx.x % 64) * V;
        if (c >= a.d) continue;
        float x[V], *y = f + g * V;
        if (a.add) load<V>(to + c, x);
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = y[e] * a.scale + (a.add ? x[e] : 0.f);
        store<V>(to + c, y);
    }
}

// The sums of whole pieces of one token.
template <class T, int V>
__global__ __launch_bounds__(256) void k_pieces(Args a) {
    constexpr int kGroups = groups<V>();
    const uint32_t piece = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / 64), lane = threadIdx.x % 64;
    const uint64_t from = (uint64_t)piece * kPiece;
    if (from + kPiece > a.n) return;
    const uint32_t id = a.ids[0][from], id_last = a.ids[0][from + kPiece - 1], held = a.at[0][from + lane % kPiece];
    if (id >= a.vocab || id_last != id) return;
    for (uint32_t c0 = 0; c0 < a.d; c0 += 64 * V * kGroups) {
        float f[kGroups * V] = {};
        add_held<T, 8, V>(a, held, 0, kPiece, c0, f);
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
            const uint32_t c = c0 + (g * 64 + lane) * V;
            if (c < a.d) store<V>(a.sums + (size_t)piece * a.d + c, f + g * V);
        }
    }
}

// A wave for every sorted position; the first of its token's run adds the run.  A run of 64 and more is added by all waves of
// the workgroup, each a share of its rows and pieces, once they are done with their own.  (Their positions follow each other, so
// no second long run begins among them.)
template <class T, class G, int V>
__global__ __launch_bounds__(256) void k_runs(Args a) {
    constexpr int kGroups = groups<V>(), kCols = 64 * V * kGroups;
    __shared__ float s_sum[3][kCols];
    __shared__ uint32_t s_begin;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const uint32_t i = min(blockIdx.x * 4 + wave, a.n - 1), here = min(i + lane, a.n - 1);
    if (threadIdx.x == 0) s_begin = a.n;
    __syncthreads();
    const auto piece_at = [&](uint32_t position) {
        return [&a, position](uint32_t j) { return a.sums + (size_t)(position / kPiece + j) * a.d; };
    };
    // one wait for all that a short run needs to know
    const uint32_t ahead = a.ids[0][here], held = a.at[0][here], previous = a.ids[0][max(i, 1u) - 1];
    const uint32_t id = __builtin_amdgcn_readfirstlane(ahead);
    if (blockIdx.x * 4 + wave < a.n && id < a.vocab && (i == 0 || previous != id)) {
        const uint32_t n = __popcll(__ballot(i + lane < a.n && ahead == id));
        if (n == 64) {
            if (lane == 0) s_begin = i;
        } else {
            const uint32_t end = i + n, first = min((i + kPiece - 1) / kPiece * kPiece, end), last = max(first, end / kPiece * kPiece);
            for (uint32_t c0 = 0; c0 < a.d; c0 += kCols) {
                float f[kGroups * V] = {};
                add_held<T, 4, V>(a, held, 0, first - i, c0, f);
                if (last > first) add_rows<2, V>((last - first) / kPiece, c0, a.d, f, piece_at(first));
                add_held<T, 4, V>(a, held, last - i, end - last, c0, f);
                write_row<G, V>(a, id, c0, f);
            }
        }
    }
    __syncthreads();
    const uint32_t begin = __builtin_amdgcn_readfirstlane(s_begin);
    if (begin == a.n) return;
    // the run's end, by 64 looks at a time ever further ahead, and then ever nearer
    const uint32_t run = a.ids[0][begin];
    uint64_t last_of = begin + 63;
    const auto equal_ahead = [&](uint64_t stride) {
        const uint64_t j = last_of + (lane + 1) * stride;
        return (uint32_t)__popcll(__ballot(j < a.n && a.ids[0][j < a.n ? j : begin] == run));
    };
    uint64_t stride = 64;
    for (;; stride *= 64) {
        const uint32_t more = equal_ahead(stride);
        last_of += more * stride;
        if (more < 64) break;
    }
    while (stride > 1) {
        stride /= 64;
        last_of += equal_ahead(stride) * stride;
    }
    const uint32_t end = (uint32_t)last_of + 1, first = (begin + kPiece - 1) / kPiece * kPiece, last = end / kPiece * kPiece;
    const uint32_t before = first - begin, pieces = (last - first) / kPiece, behind = end - last;
    const uint32_t held0 = a.at[0][min(begin + lane, a.n - 1)], held1 = a.at[0][min(last + lane, a.n - 1)];
    const auto share = [&](uint32_t n, uint32_t w) { return (uint32_t)((uint64_t)n * w / 4); };
    for (uint32_t c0 = 0; c0 < a.d; c0 += kCols) {
        float f[kGroups * V] = {};
        uint32_t from = share(before, wave);
        add_held<T, 4, V>(a, held0, from, share(before, wave + 1) - from, c0, f);
        from = first / kPiece + share(pieces, wave);
        add_rows<4, V>(share(pieces, wave + 1) - share(pieces, wave), c0, a.d, f, piece_at(from * kPiece));
        const uint32_t rest = share(behind, wave);
        add_held<T, 4, V>(a, held1, rest, share(behind, wave + 1) - rest, c0, f);
        if (wave)
#pragma unroll
            for (int e = 0; e < kGroups * V; e++) s_sum[wave - 1][e * 64 + lane] = f[e];
        __syncthreads();
        if (!wave) {
#pragma unroll
            for (int w = 0; w < 3; w++)
#pragma unroll
                for (int e = 0; e < kGroups * V; e++) f[e] += s_sum[w][e * 64 + lane];
            write_row<G, V>(a, run, c0, f);
        }
        __syncthreads();
    }
}

// Few tokens without a sort: a workgroup for every position looks for its token in all of them, ends if it stands at an earlier
// one, and adds the rows of those where it stands: each of its waves 64 V kGroups channels, or where there are many, each a
// part of the rows.  (701 tokens of 1,101 channels: 9 us.  Sorted by one workgroup 15, and 30 for pieces and runs.)
template <class T, class G, int V>
__global__ __launch_bounds__(256) void k_few(Args a) {
    constexpr int kRounds = kFew / 64, kGroups = kFewGroups, kCols = 64 * V * kGroups;
    __shared__ uint32_t s_at[kFew];
    __shared__ float s_sum[3][kCols];
    const uint32_t i = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const uint32_t id = id_of(a, i);
    if (id >= a.vocab) return;
    uint32_t n = 0;
    bool earlier = false;
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        const uint32_t j = r * 64 + lane;
        if (r * 64u < a.n) {
            const bool same = j < a.n && id_of(a, min(j, a.n - 1)) == id;
            const uint64_t all = __ballot(same);
            earlier |= __ballot(same && j < i) != 0;
            if (same && wave == 0) s_at[n + __popcll(all & ((1ull << lane) - 1))] = j;
            n += __popcll(all);
        }
    }
    if (earlier) return;  // in all waves alike
    __syncthreads();
    const auto row = [&](uint32_t j) {
        return (const T*)a.from + (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane(s_at[j]) * a.from_stride;
    };
    const uint32_t c_from = blockIdx.y * 4 * kCols, c_to = min(a.d, c_from + 4 * kCols);
    const bool split = n > 16;
    const uint32_t j0 = split ? n * wave / 4 : 0, j1 = split ? n * (wave + 1) / 4 : n;
    for (uint32_t c0 = c_from + (split ? 0 : wave * kCols); c0 < c_to; c0 += split ? kCols : 4 * kCols) {
        float f[kGroups * V] = {};
        add_rows<8, V>(j1 - j0, c0, a.d, f, [&](uint32_t j) { return row(j0 + j); });
        if (split) {
            if (wave)
#pragma unroll
                for (int e = 0; e < kGroups * V; e++) s_sum[wave - 1][e * 64 + lane] = f[e];
            __syncthreads();
            if (!wave)
#pragma unroll
                for (int w = 0; w < 3; w++)
#pragma unroll
                    for (int e = 0; e < kGroups * V; e++) f[e] += s_sum[w][e * 64 + lane];
            __syncthreads();
            if (wave) continue;
        }
        write_row<G, V>(a, id, c0, f);
    }
}

int check(const fhe_ssm_embedding* a) {
    if (!a) return fail(CKKS_EINVAL, "embedding: null description");
    if (a->table_type > FHE_SSM_F16 || a->row_type > FHE_SSM_F16) return fail(CKKS_EINVAL, "embedding: unknown type");
    if (a->vocab < 1 || a->vocab > kMostVocab) return fail(CKKS_EINVAL, "embedding: a vocabulary of %u", a->vocab);
    if (a->channels < 1 || a->channels > 1u << 20) return fail(CKKS_EINVAL, "embedding: %u channels", a->channels);
    if (a->tokens > kMostTokens) return fail(CKKS_EINVAL, "embedding: too many tokens");
    return CKKS_OK;
}

struct Layout {
    uint32_t bits[2], tiles, parts;
    size_t ids[2], at[2], counts, sums, bytes;
};
Layout layout(const fhe_ssm_embedding& a) {
    Layout y{};
    uint32_t bits = 1;
    while (a.vocab >> bits) bits++;  // of the vocabulary's size itself, which stands for tokens outside
    y.bits[0] = (bits + 1) / 2, y.bits[1] = std::max(1u, bits / 2);
    const uint32_t tiles = (a.tokens + kTile - 1) / kTile;
    y.tiles = std::max(1u, (tiles + kMostParts - 1) / kMostParts);
    y.parts = (tiles + y.tiles - 1) / y.tiles;
    const bool small = a.tokens <= kSmall;
    const auto put = [&](size_t n) {
        const size_t at = y.bytes;
        y.bytes += (n + 255) / 256 * 256;
        return at;
    };
    if (a.tokens <= kFew) return y;
    const size_t list = a.tokens * sizeof(uint32_t);
    y.ids[0] = put(list), y.at[0] = put(list);
    y.ids[1] = put(small ? 0 : list), y.at[1] = put(small ? 0 : list);
    y.counts = put(small ? 0 : (size_t)y.parts * kDigits * sizeof(uint32_t));
    y.sums = put((size_t)(a.tokens / kPiece) * a.channels * sizeof(float));
    return y;
}

bool on_vectors(const void* p, int64_t stride, size_t size, int v) { return aligned(p, size * v) && stride % v == 0; }

}  // namespace
}  // namespace clear

extern "C" {

int fhe_ssm_embedding_lookup(const fhe_ssm_embedding* a, const int64_t* tokens, const void* table, void* out, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (a->tokens == 0) return CKKS_OK;
    if (!tokens || !table || !out) return fail(CKKS_EINVAL, "embedding: null argument");
    if (a->table_stride < (int64_t)a->channels) return fail(CKKS_EINVAL, "embedding: rows of the table overlap");
    if (a->tokens > 1 && a->row_stride < (int64_t)a->channels) return fail(CKKS_EINVAL, "embedding: output rows overlap");
    Args k{};
    k.tokens = tokens, k.from = table, k.to = out, k.n = a->tokens, k.vocab = a->vocab, k.d = a->channels;
    k.from_stride = a->table_stride, k.to_stride = a->tokens > 1 ? a->row_stride : 0, k.scale = a->scale;
    return by_type(a->table_type, [&](auto f) {
        return by_type(a->row_type, [&](auto t) {
            typedef decltype(f) F;
            typedef decltype(t) T;
            constexpr int V = 16 / (sizeof(F) > sizeof(T) ? sizeof(F) : sizeof(T));
            const bool vectors = k.d % V == 0 && on_vectors(table, k.from_stride, sizeof(F), V) && on_vectors(out, k.to_stride, sizeof(T), V);
            const auto run = [&](auto v) {
                constexpr int kV = decltype(v)::value;
                const uint32_t vectors = (k.d + kV - 1) / kV;
                const uint64_t all = vectors < 256 ? ((uint64_t)k.n * vectors + 1023) / 1024 : (uint64_t)k.n * ((vectors + 1023) / 1024);
                const dim3 blocks((uint32_t)std::min<uint64_t>(all, 1u << 22));
                if (vectors < 256) hipLaunchKernelGGL((k_lookup<F, T, kV>), blocks, dim3(256), 0, (hipStream_t)stream, k);
                else hipLaunchKernelGGL((k_lookup_long<F, T, kV>), blocks, dim3(256), 0, (hipStream_t)stream, k);
                return launched("embedding");
            };
            return vectors ? run(std::integral_constant<int, V>{}) : run(std::integral_constant<int, 1>{});
        });
    });
}

int fhe_ssm_embedding_workspace(const fhe_ssm_embedding* a, size_t* bytes) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (!bytes) return fail(CKKS_EINVAL, "embedding: null argument");
    *bytes = layout(*a).bytes;
    return CKKS_OK;
}

int fhe_ssm_embedding_gradient(const fhe_ssm_embedding* a, const int64_t* tokens, const void* dout, void* dtable,
                               int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace clear;
    if (int rc = check(a)) return rc;
    if (!dtable || (a->tokens && (!tokens || !dout))) return fail(CKKS_EINVAL, "embedding: null argument");
    if (a->table_type != FHE_SSM_F32 && a->table_type != a->row_type)
        return fail(CKKS_EINVAL, "embedding: the table's gradient is float32 or of the rows' type");
    if (!aligned(dtable, type_bytes(a->table_type))) return fail(CKKS_EINVAL, "embedding: the table's gradient lies between elements");
    if (a->tokens > 1 && a->row_stride < 0) return fail(CKKS_EINVAL, "embedding: a negative stride");
    const Layout y = layout(*a);
    if (y.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < y.bytes))
        return fail(CKKS_EINVAL, "embedding: the workspace must have %zu bytes and lie on 16", y.bytes);
    Args k{};
    k.tokens = tokens, k.from = dout, k.to = dtable, k.n = a->tokens, k.vocab = a->vocab, k.d = a->channels;
    k.from_stride = a->tokens > 1 ? a->row_stride : 0, k.scale = a->scale, k.add = accumulate != 0;
    k.tiles = y.tiles, k.parts = y.parts;
    uint8_t* w = (uint8_t*)workspace;
    for (int i = 0; i < 2; i++) k.bits[i] = y.bits[i], k.ids[i] = (uint32_t*)(w + y.ids[i]), k.at[i] = (uint32_t*)(w + y.at[i]);
    k.counts = (uint32_t*)(w + y.counts), k.sums = (float*)(w + y.sums);
    const hipStream_t st = (hipStream_t)stream;
    const size_t table = (size_t)a->vocab * a->channels * type_bytes(a->table_type);
    const size_t head = std::min(table, (16 - (uintptr_t)dtable % 16) % 16), words = (table - head) / 16, tail = table - head - 16 * words;
    k.zero_at = (u32x4*)((uint8_t*)dtable + head);
    k.edge[0] = (uint16_t*)dtable, k.edges[0] = (uint32_t)(head / 2);
    k.edge[1] = (uint16_t*)(k.zero_at + words), k.edges[1] = (uint32_t)(tail / 2);
    // the kernels of the sort, each with its share of the table beside it; two workgroups of them fit a CU
    const bool small = k.n <= kSmall;
    if (!k.n && k.add) return CKKS_OK;
    const auto sort = [&](auto kernel, int i, int of, uint32_t parts) {
        k.zero_blocks = k.add ? 0 : (uint32_t)std::min<size_t>(512, words / of / 4096 + 1);
        k.zero_from = words * i / of, k.zero_to = words * (i + 1) / of;
        hipLaunchKernelGGL(kernel, dim3(parts + k.zero_blocks), dim3(1024), 0, st, k);
    };
    const bool few = k.n <= kFew;
    if (few) {
        if (!k.add) sort(k_zero, 0, 1, 0);
    } else if (k.n <= 2048) sort(k_sort_small<2>, 0, 1, 1);
    else if (k.n <= 4096) sort(k_sort_small<4>, 0, 1, 1);
    else if (small) sort(k_sort_small<8>, 0, 1, 1);
    else {
        sort(k_count<0>, 0, 4, k.parts);
        sort(k_move<0>, 1, 4, k.parts);
        sort(k_count<1>, 2, 4, k.parts);
        sort(k_move<1>, 3, 4, k.parts);
    }
    if (int rc = launched("embedding: sorting the tokens")) return rc;
    if (!k.n) return CKKS_OK;
    return by_type(a->row_type, [&](auto t) {
        typedef decltype(t) T;
        const auto add = [&](auto g, auto v) {
            typedef decltype(g) G;
            constexpr int V = decltype(v)::value;
            if (few) {
                hipLaunchKernelGGL((k_few<T, G, V>), dim3(k.n, (k.d + 256 * V * kFewGroups - 1) / (256 * V * kFewGroups)), dim3(256), 0, st, k);
                return launched("embedding: gradient");
            }
            if (k.n >= kPiece) hipLaunchKernelGGL((k_pieces<T, V>), dim3((k.n / kPiece + 3) / 4), dim3(256), 0, st, k);
            hipLaunchKernelGGL((k_runs<T, G, V>), dim3((k.n + 3) / 4), dim3(256), 0, st, k);
            return launched("embedding: gradient");
        };
        constexpr int kWide = 16 / sizeof(T);
        const std::integral_constant<int, kWide> wide;
        const std::integral_constant<int, 1> one;
        const bool vectors = k.d % kWide == 0 && on_vectors(dout, k.from_stride, sizeof(T), kWide) &&
                             aligned(dtable, kWide * type_bytes(a->table_type));
        if (a->table_type == FHE_SSM_F32) return vectors ? add(0.f, wide) : add(0.f, one);
        return vectors ? add(T{}, wide) : add(T{}, one);
    });
}

}  // extern "C"
