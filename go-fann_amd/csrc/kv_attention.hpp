// kv_attention.hpp -- attention over the paged 4-bit key/value cache, and the
// join of its partial results.
#pragma once

#include "kv_common.hpp"

namespace gofann {
namespace kv {

struct AttendArgs {
    Batch batch;
    Rows q, out;
    const uint8_t* k_codes;
    const uint8_t* k_scales;
    const uint8_t* v_codes;
    const uint8_t* v_scales;
    const int32_t* blocks;  // [queries][kv_heads][width] or NULL
    float* lse;             // [queries][heads] or NULL
    float* part_o;          // [kv_heads][split][part_count][dim], splits > 1: see part_of()
    float* part_ml;         // [kv_heads][split][part_count][2]: reference, sum
    int32_t* pieces;        // [row tile][kv_heads][2] of shared tiles: first slot, shares after it
    const uint32_t* live;   // [sequence][live_stride][4]: tiles that the filter leaves, as kv_live_kernel
    const int32_t* live_count;  // kv_live_kernel; NULL: all of them are looked at
    int64_t live_stride;
    int join_shift;         // log2 of the groups of lanes that join a row's pieces
    uint32_t* arrived;      // [item], zero between calls: splits done; NULL: kv_join_kernel joins
    float scale_log2;       // scale * log2(e)
    int group;              // heads a key/value head
    int width;
    int row_tiles;          // row tiles of a sequence (listed: of a token times tokens)
    int token_tiles;        // listed: row tiles of one token's heads
    int splits;
    int split_tiles;        // tiles of a split
    int rows_over;          // sequences of at most so many rows are not this launch's,
    int rows_upto;          // nor those of more than so many
    int64_t part_count;     // rows with partial results: the call's, or of every
    int part_rows;          // sequence so many where that is not 0
    int slots;              // row tiles counted through the sequences; 0: a grid of them
    int sequences;
    const uint32_t* sees;   // kDraft: [queries][sees_stride] words, sees_width used
    int64_t sees_stride;
    int sees_width;
};

// Which positions a token may look at, the filter apart: those up to its own;
// those before its sequence's tokens and of these the ones that its `sees` bits
// name; or all of a sequence that it is no part of.  Each is compiled by itself,
// so that the first has nothing to carry for the others.
enum Reach { kOwn = 0, kDraft = 1, kCross = 2 };

// What a workgroup works on: row tile `index` of sequence b, the id-th of all.
struct Item {
    int b, index;
    int64_t id;
};

// Row tiles of a sequence are blockIdx.y, sequences blockIdx.z.  Where sequences
// differ so much in their tokens that most of that grid would find nothing, the
// tiles are counted through them instead (slots): those of sequence b begin at
// offset[b] group / rows + b, which leaves each room for its last, part tile
// (listed: at its first token's), so that a search of the offsets is all that
// is needed.  False: no such tile.
__device__ __forceinline__ bool item_of(const AttendArgs& a, int rows, Item& it)
{
    const Batch& t = a.batch;
    if (a.slots == 0) {
        it.b = blockIdx.z;
        it.index = gridDim.y - 1 - blockIdx.y;  // the longest rows first
        it.id = static_cast<int64_t>(it.b) * a.row_tiles + it.index;
        return true;
    }
    const int64_t from_end = static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y;
    it.id = a.slots - 1 - from_end;
    if (it.id < 0) return false;
    const auto begin = [&](int b) {
        const int64_t q0 = t.first_query(b);
        return a.blocks != nullptr ? q0 * a.token_tiles : q0 * a.group / rows + b;
    };
    // The last sequence that begins no later: 64 are looked at in each round.
    const int lane = threadIdx.x % 64;
    int b = 0, count = a.sequences;
    while (count > 1) {
        const int step = (count + 63) / 64;
        const int at = lane * step;
        const int below = __popcll(__ballot(at < count && begin(b + (at < count ? at : 0)) <= it.id));
        const int skip = below > 0 ? (below - 1) * step : 0;
        b += skip;
        count = count - skip < step ? count - skip : step;
    }
    it.b = __builtin_amdgcn_readfirstlane(b);
    const int q0 = t.first_query(it.b);
    const int64_t n = t.new_tokens(it.b, q0);
    const int64_t index = it.id - begin(it.b);
    const int64_t tiles = a.blocks != nullptr ? n * a.token_tiles : (n * a.group + rows - 1) / rows;
    if (index < 0 || index >= tiles) return false;
    it.index = static_cast<int>(index);
    return true;
}

// Where the partial results of a sequence's first row lie, in rows: a tile's
// rows lie together, as they are written (with a row's splits together instead,
// 19 sequences of five tokens and four heads a group took 26.1 us, not 25.2).
__device__ __forceinline__ int64_t part_of(const AttendArgs& a, int b, int q0, int h, int split)
{
    const int64_t first = a.part_rows > 0 ? static_cast<int64_t>(b) * a.part_rows
                                          : static_cast<int64_t>(q0) * a.group;
    return (static_cast<int64_t>(h) * a.splits + split) * a.part_count + first;
}

// The rows of one row tile: rows [begin, end) of the sequence's flattened
// (token, head of the group) rows, and the positions they reach.
struct RowTile {
    int begin, end;
    int first_pos;            // the last that every row sees: the first row's token's
    int last_pos;             // the last that any row sees, or that may have a page
    int token;                // listed: the one token
};

template <int kReach>
__device__ __forceinline__ RowTile row_tile(const AttendArgs& a, int index, int rows, int len, int n)
{
    RowTile t;
    if (a.blocks != nullptr) {
        t.token = index / a.token_tiles;
        t.begin = t.token * a.group + (index % a.token_tiles) * rows;
        t.end = (t.token + 1) * a.group;
        if (t.token >= n) t.end = t.begin;
    } else {
        t.token = 0;
        t.begin = index * rows;
        t.end = n * a.group;
    }
    if (n * a.group <= a.rows_over || n * a.group > a.rows_upto) t.end = t.begin;
    if (t.end > t.begin + rows) t.end = t.begin + rows;
    if constexpr (kReach == kOwn) {
        t.first_pos = len - n + t.begin / a.group;
        t.last_pos = len - n + (t.end - 1) / a.group;
    } else {
        t.first_pos = kReach == kDraft ? len - n - 1 : len - 1;
        t.last_pos = len - 1;
    }
    if (t.last_pos >= a.batch.max_positions) t.last_pos = a.batch.max_positions - 1;
    return t;
}

// How far, in powers of two, a score may pass the running maximum before that
// is renewed.  The reference m that weights are taken against lies E::kRaise
// below it, so weights reach 2^(kSlack + kRaise): with 0 for bf16 and 7 for f16,
// whose weights would otherwise lose, below 2^-25, a tail of many small ones.
constexpr float kSlack = 8.0f;

// References past this are multiples of 1/2 and more, and a score's weight would
// be that of its exact product against a rounded one, off by powers of two (from
// 2^31 on zeros and infinities).  There the products are rounded as the
// reference was, in the way of a renewal: chunks of 2,048 tokens take 1% longer
// for it, single tokens what they did.
constexpr float kFar = 4194304.0f;

// Splits up to which the last workgroup of an item to finish joins them
// itself; past it the partial results are too many for one workgroup.
constexpr int kJoinSplits = 16;

// Partial results go between workgroups of one launch as accesses of device
// scope, eight bytes at a time.
__device__ __forceinline__ void put2(float* p, float x, float y)
{
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, float2{x, y}),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p)
{
    return __builtin_bit_cast(
        float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                  __HIP_MEMORY_SCOPE_AGENT));
}

// Tiles of 32 positions that a row tile reads.
__device__ __forceinline__ int tiles_of(const AttendArgs& a, const RowTile& t)
{
    if (t.end <= t.begin || t.last_pos < 0) return 0;
    if (a.blocks != nullptr) return a.width << (a.batch.page_shift - 5);
    return (t.last_pos >> 5) + 1;
}

// Four channels of a row's output, from the weighted values and the weights'
// sum in units of 2^top.
template <class E>
__device__ __forceinline__ void finish(const AttendArgs& a, const Batch& t, int q0, int h, int row,
                                       int ch, f32x4 acc, float top, float total)
{
    const int token = q0 + row / a.group, head = h * a.group + row % a.group;
    uint16_t* const to = a.out.p + token * a.out.token_stride + head * a.out.head_stride + ch;
    const float inv = total != 0.0f ? 1.0f / total : 0.0f;
    typename E::V2 lo, hi;
    lo[0] = static_cast<typename E::T>(acc[0] * inv);
    lo[1] = static_cast<typename E::T>(acc[1] * inv);
    hi[0] = static_cast<typename E::T>(acc[2] * inv);
    hi[1] = static_cast<typename E::T>(acc[3] * inv);
    u32x2 v{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    // One rounding for both ways of storing: moved into the branches, one of
    // them would become a product and conversion in a single instruction.
    asm("" : "+v"(v));
    if (a.out.wide) {
        *reinterpret_cast<u32x2*>(to) = v;
    } else {
        to[0] = static_cast<uint16_t>(v[0]);
        to[1] = static_cast<uint16_t>(v[0] >> 16);
        to[2] = static_cast<uint16_t>(v[1]);
        to[3] = static_cast<uint16_t>(v[1] >> 16);
    }
    if (a.lse != nullptr && ch == 0)
        a.lse[static_cast<int64_t>(token) * t.kv_heads * a.group + head] =
            (top + __builtin_log2f(total)) * 0.69314718055994531f;
}

// Scores of a lane's eight positions, -inf where the row may not look: bit e
// of `mine` is position e's, and only the first `left` are before the row's end.
__device__ __forceinline__ void mask_scores(f32x4 (&s)[2], uint32_t mine, int left)
{
    left = left < 0 ? 0 : left > 8 ? 8 : left;
    const uint32_t ok = mine & ((1u << left) - 1u);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e / 4][e % 4] = (ok >> e & 1u) ? s[e / 4][e % 4] : -__builtin_inff();
}

// The bits of a draft's token (row `row` of `sees`) for the 32 positions that
// begin `rel` past the draft's first: positions before that are all seen.  Two
// words, loaded ahead of their use.
struct Sees {
    uint32_t lo, hi;
};
__device__ __forceinline__ Sees load_sees(const AttendArgs& a, int row, int rel)
{
    Sees s{0, 0};
    const int w = rel >> 5;
    const uint32_t* const p = a.sees + static_cast<int64_t>(row) * a.sees_stride;
    if (row >= 0 && w >= 0 && w < a.sees_width) s.lo = p[w];
    if (row >= 0 && w >= -1 && w + 1 < a.sees_width) s.hi = p[w + 1];
    return s;
}
__device__ __forceinline__ uint32_t sees_bits(Sees s, int row, int rel)
{
    uint32_t v = __builtin_amdgcn_alignbit(s.hi, s.lo, rel & 31);
    if (rel < 0) v |= rel <= -32 ? 0xFFFFFFFFu : (1u << -rel) - 1u;
    return row < 0 ? 0u : v;
}

// The scale of a position that was never written may be anything, and a weight
// of zero times an infinity or NaN is NaN: exponents that append writes to no
// group become 1.
template <class E>
__device__ __forceinline__ uint32_t written_scale(uint32_t scale)
{
    const uint32_t e = scale >> 23 & 255u;
    return e - (127 + E::kMinExp) <= static_cast<uint32_t>(E::kMaxExp - E::kMinExp) ? scale : 127u << 23;
}

// A row's softmax so far.
struct Row {
    float m = -__builtin_inff();  // the reference: weights are 2^(scaled score - m)
    float mu = 0.0f;              // m, or 0 while there is none or it is past kFar
    float sum = 0.0f;             // of the weights
};

// The reference renewed by a tile's scaled maximum; returns the factor of what
// was summed so far.  is_far: it is past kFar, to be taken off by far_score().
template <class E>
__device__ __forceinline__ float renew(Row& w, float top, bool& is_far)
{
    const float fresh = fmaxf(w.m, top - E::kRaise);
    const float keep = fresh == -__builtin_inff() ? 0.0f : fresh;
    const float f = __builtin_amdgcn_exp2f(w.m - keep);
    is_far = __builtin_fabsf(keep) > kFar && __builtin_fabsf(keep) < __builtin_inff();
    w.m = fresh;
    w.mu = is_far ? 0.0f : keep;
    w.sum *= f;
    return f;
}

// A score whose scaled value is less by the reference.
__device__ __forceinline__ float far_score(float s, float scale_log2, float m)
{
    return (s * scale_log2 - m) * __builtin_amdgcn_rcpf(scale_log2);
}

// Weights 2^(score - m) of a row's scores, the row's statistics and weighted
// values o brought along; far: a row of the wave has a reference past kFar, and
// all tiles go the way of a renewal.  The reference is renewed only where a
// score passes the maximum it was made from by more than kSlack (in powers of
// two): until then the weights are at most 2^(kSlack + kRaise), which costs
// 32-bit sums nothing.  The weights enter the product in 16 bits, as the values
// do; their sum stays in 32.
template <class E, int kUnit>
__device__ __forceinline__ typename E::V8 weigh(f32x4 (&s)[2], float scale_log2, Row& row, bool& far,
                                                f32x4 (&o)[kUnit])
{
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e / 4][e % 4]);
    top *= scale_log2;
    if (far || __any(top - row.m > kSlack + E::kRaise)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        bool mine;
        const float f = renew<E>(row, top, mine);
#pragma unroll
        for (int c = 0; c < kUnit; ++c) o[c] *= f;
        far = __any(mine);
        if (mine) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e / 4][e % 4] = far_score(s[e / 4][e % 4], scale_log2, row.m);
        }
    }
    typename E::V8 p;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e / 4][e % 4], scale_log2, -row.mu));
        row.sum += w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = static_cast<typename E::T>(w[e]);
    return p;
}

// What a lane loads of one tile: keys of two positions, values of eight.
template <int D>
struct Raw {
    static constexpr int kGroups = D == 256 ? 2 : 1;
    uint32_t k[2][D / 32];
    uint32_t ks[2][kGroups];
    uint32_t v[D / 16];
    uint32_t vs[2];
};

// What a workgroup works on: tiles [begin, end) of a row tile.
struct Piece {
    int b, h, len, q0, n;
    int begin, end;
    int slot;  // of its partial result; negative: it has all of the row tile
    RowTile rows;
};

// Where the four waves of a workgroup of few rows join what they have.
template <int D, int NT>
struct FewLds {
    static constexpr int kResident = NT == 2 && D == 256 ? 1 : NT == 2 || D == 256 ? 2 : D == 128 ? 4 : 5;
    float m[4][16 * NT], sum[4][16 * NT];
    __attribute__((aligned(16))) float o[4][16][D + 4];  // rows start on other banks
};

// One row tile of one key/value head over one split of its positions.
//
// A tile of 32 positions is two 16 x 16 score tiles S^T = K Q^T and D / 16
// product tiles O^T += V^T P^T, all v_mfma_f32_16x16x32.  The order of the
// contracted index is free as long as both operands agree, and is chosen so
// that nothing crosses lanes: lane (r, g) = (lane % 16, lane / 16)
//   * holds, as rows of S^T, keys 8 (r / 4) + r % 4 and that plus 4, whose
//     channels [g dim/4, ..) are one or two 16-byte loads under one scale;
//   * gets the scores of query r against the eight positions 8 g .. 8 g + 7,
//     which are just the eight slots of P^T that lane (r, g) feeds;
//   * holds, as rows of V^T, the dim / 16 channels of unit r at those eight
//     positions, one run of dim / 4 bytes in the cache;
//   * ends with the channels [g dim/4, (g+1) dim/4) of query r's output.
// The 4-bit codes become 16-bit elements by the hardware's conversion, which
// applies the group's power of two; both are exact.
//
// Four waves take every fourth tile each and are joined through LDS; splits of
// the positions fill the chip where there are few rows.  HBM bounds long calls:
// one token of 64 heads over 500,001 positions (544 MB) takes 98 us, 5.6 TB/s
// (a large copy, read and written: 4.8), and 11 us for the join of 96 splits.
// At 128 channels it has 128 registers and four workgroups resident a CU; with
// three, and masked tiles not yet loaded ahead, sequences of 500 to 16,000
// positions took 9% longer.  64 channels: five; 256: two, by 201 registers and
// by the 69 KB of LDS that join the waves.  Short calls are a chain of dependent
// loads: 8.6 us for 1,999 positions of 8 heads.
template <class E, int D, int kReach, int NT, class F>
__device__ __forceinline__ void few_rows(const AttendArgs& a, FewLds<D, NT>& lds, const Piece& piece, F&& put)
{
    using V8 = typename E::V8;
    constexpr int kUnit = D / 16;  // channels of a unit, tiles of O
    const Batch& t = a.batch;
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int r16 = lane % 16, g4 = lane / 16;
    const int h = piece.h, b = piece.b, len = piece.len, q0 = piece.q0, n = piece.n;
    const RowTile& rt = piece.rows;
    const int tile_begin = piece.begin, tile_end = piece.end;
    const int hi_pos = rt.last_pos + 1;                         // positions that are read
    const int all_see = rt.first_pos + 1;                       // positions that every row sees

    // The rows' queries and limits: positions that they see, or, of a draft's
    // tokens, the row of their bits (-1: not a row).
    V8 q[NT][D / 32];
    int limit[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = rt.begin + 16 * nt + r16;
        const bool in = row < rt.end;
        const int i = (in ? row : rt.begin) / a.group;
        const int head = h * a.group + (in ? row : rt.begin) % a.group;
        limit[nt] = kReach == kDraft ? (in ? q0 + i : -1) : !in ? 0 : kReach == kCross ? len : len - n + i + 1;
        const uint16_t* const p = a.q.p + (q0 + i) * a.q.token_stride + head * a.q.head_stride;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            // Channels that the dword j of a lane's keys holds.
            const int c = D == 64 ? 16 * g4 + 8 * j : 128 * (j / 4) + 32 * g4 + 8 * (j % 4);
            q[nt][j] = __builtin_bit_cast(V8, load8(p + c, a.q.wide));
        }
    }

    f32x4 o[NT][kUnit];
    Row st[NT];
    bool far[NT] = {};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < kUnit; ++c) o[nt][c] = f32x4{0, 0, 0, 0};
    }

    // Keys and values of tile `at`, loaded apart: a tile's keys are requested
    // once the last tile's scores are formed, its values once the last tile's
    // product is, each into the registers just freed.
    Raw<D> x;
    const auto load_keys = [&](uint32_t at) {
        const uint8_t* const kc = a.k_codes + static_cast<uint64_t>(at) * (16 * D);
        const uint8_t* const ks = a.k_scales + static_cast<uint64_t>(at) * D;
        const uint32_t pos = 8 * (r16 / 4) + r16 % 4;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t p = pos + 4 * s;
            if constexpr (D == 64) {
                const u32x2 v = *reinterpret_cast<const u32x2*>(kc + p * (D / 2) + 8 * g4);
                x.k[s][0] = v[0];
                x.k[s][1] = v[1];
                x.ks[s][0] = ks[p * (D / 32) + g4 / 2];
            } else {
#pragma unroll
                for (int c = 0; c < D / 128; ++c) {
                    const u32x4 v = *reinterpret_cast<const u32x4*>(kc + p * (D / 2) + 64 * c + 16 * g4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x.k[s][4 * c + j] = v[j];
                    x.ks[s][c] = ks[p * (D / 32) + 4 * c + g4];
                }
            }
        }
    };
    const auto load_values = [&](uint32_t at) {
        const uint8_t* const vc = a.v_codes + static_cast<uint64_t>(at) * (16 * D);
        const uint8_t* const vs = a.v_scales + static_cast<uint64_t>(at) * D;
        const uint8_t* const vp = vc + (g4 * 16 + r16) * (D / 4);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(vp + 16 * c);
#pragma unroll
            for (int j = 0; j < 4; ++j) x.v[4 * c + j] = v[j];
        }
        const u32x2 s = *reinterpret_cast<const u32x2*>(vs + (g4 * (D / 32) + r16 * kUnit / 32) * 8);
        x.vs[0] = s[0];
        x.vs[1] = s[1];
    };

    f32x4 s[NT][2];
    const auto scores = [&]() {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][half] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const uint32_t sc = x.ks[half][D == 256 ? j / 4 : 0] << 23;
                const uint32_t c = x.k[half][j];
                const u32x4 e{E::template decode<0>(c, sc), E::template decode<1>(c, sc),
                              E::template decode<2>(c, sc), E::template decode<3>(c, sc)};
                const V8 k8 = __builtin_bit_cast(V8, e);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][half] = E::mfma(k8, q[nt][j], s[nt][half]);
            }
        }
    };
    V8 p[NT];
    uint32_t scale[8];  // of the eight positions' values, in bits 30:23
    const auto value_scales = [&]() {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            scale[4 * w] = x.vs[w] << 23;
            scale[4 * w + 1] = x.vs[w] << 15;
            scale[4 * w + 2] = x.vs[w] << 7;
            scale[4 * w + 3] = x.vs[w] >> 1;
        }
    };
    // Two positions' bytes to pairs of channels, then to pairs of positions a
    // channel.
    const auto product = [&]() {
        each<kUnit / 2>([&](auto pair) {
            constexpr int c = decltype(pair)::value;  // channels 2 c, 2 c + 1 of the unit
            uint32_t d[8];
            each<8>([&](auto pos) {
                constexpr int e = decltype(pos)::value;
                constexpr int byte = e * (D / 32) + c;
                d[e] = E::template decode<byte % 4>(x.v[byte / 4], scale[e]);
            });
            u32x4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                even[j] = __builtin_amdgcn_perm(d[2 * j + 1], d[2 * j], 0x05040100u);
                odd[j] = __builtin_amdgcn_perm(d[2 * j + 1], d[2 * j], 0x07060302u);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][2 * c] = E::mfma(__builtin_bit_cast(V8, even), p[nt], o[nt][2 * c]);
                o[nt][2 * c + 1] = E::mfma(__builtin_bit_cast(V8, odd), p[nt], o[nt][2 * c + 1]);
            }
        });
    };

    // This wave's tiles, 64 at a time: lane l looks up the l-th one's page and
    // filter word, so that only tiles with a visible position are visited and
    // the next one's address is at hand while it is loaded.
    const int page_tiles_shift = t.page_shift - 5;
    for (int base = tile_begin + wave; base < tile_end; base += 64 * 4) {
        const int tile = base + lane * 4;
        uint32_t at = 0, word = 0;
        int t0 = 0;
        if (tile < tile_end) {
            if (kReach != kOwn && a.live != nullptr) {
                const u32x4 entry = reinterpret_cast<const u32x4*>(a.live)[b * a.live_stride + tile];
                const int page = entry[2];
                t0 = static_cast<int>(entry[0]) * kTile;
                if (page >= 0) {
                    word = entry[1];
                    at = ((static_cast<uint32_t>(page) * t.kv_heads + h) << page_tiles_shift) +
                         (entry[0] & ((1 << page_tiles_shift) - 1));
                }
            } else {
                int block = tile >> page_tiles_shift;
                const int within = tile & ((1 << page_tiles_shift) - 1);
                if (a.blocks != nullptr)
                    block = a.blocks[(static_cast<int64_t>(q0 + rt.token) * t.kv_heads + h) * a.width + block];
                const int page = t.page(b, block);
                // A block of a list may lie anywhere: only positions below hi_pos count.
                if (page >= 0 && block <= (rt.last_pos >> t.page_shift)) {
                    t0 = (block << t.page_shift) + kTile * within;
                    if (t0 < hi_pos) {
                        word = t.word(b, t0 >> 5);
                        if (hi_pos - t0 < 32) word &= (1u << (hi_pos - t0)) - 1u;
                        at = ((static_cast<uint32_t>(page) * t.kv_heads + h) << page_tiles_shift) + within;
                    }
                }
            }
        }
        // Tiles that every row sees whole, then the others.
        uint64_t whole = __ballot(word == 0xFFFFFFFFu && t0 + kTile <= all_see);
        uint64_t part = __ballot(word != 0) & ~whole;
        const auto run = [&](auto kind, uint64_t live) {
            constexpr bool kMasked = decltype(kind)::value;
            if (live == 0) return;
            int i = __builtin_ctzll(live);
            load_keys(__builtin_amdgcn_readlane(at, i));
            load_values(__builtin_amdgcn_readlane(at, i));
            while (true) {
                live &= live - 1;
                const bool more = live != 0;
                const int next = more ? __builtin_ctzll(live) : i;
                const uint32_t ahead = __builtin_amdgcn_readlane(at, next);
                const int first = __builtin_amdgcn_readlane(t0, i);
                [[maybe_unused]] const int rel = first - (len - n);
                [[maybe_unused]] Sees sees[NT];
                if constexpr (kMasked && kReach == kDraft) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) sees[nt] = load_sees(a, limit[nt], rel);
                }
                scores();
                if (more) load_keys(ahead);
                uint32_t mine = 0;
                if constexpr (kMasked) {
                    mine = static_cast<uint32_t>(__builtin_amdgcn_readlane(word, i)) >> (8 * g4);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if constexpr (kReach == kDraft)
                            mask_scores(s[nt], mine & sees_bits(sees[nt], limit[nt], rel) >> (8 * g4), 8);
                        else
                            mask_scores(s[nt], mine, limit[nt] - (first + 8 * g4));
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    p[nt] = weigh<E, kUnit>(s[nt], a.scale_log2, st[nt], far[nt], o[nt]);
                value_scales();
                if constexpr (kMasked) {
                    // A position that no row sees may hold anything: its scale
                    // must not turn a weight of zero into a NaN.
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (!(mine >> e & 1u)) scale[e] = 127u << 23;
                        if constexpr (kReach == kDraft) scale[e] = written_scale<E>(scale[e]);
                    }
                }
                product();
                if (!more) break;
                load_values(ahead);
                i = next;
            }
        };
        run(std::false_type{}, whole);
        run(std::true_type{}, part);
    }

#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        st[nt].sum += __shfl_xor(st[nt].sum, 16);
        st[nt].sum += __shfl_xor(st[nt].sum, 32);
    }

    // The four waves' maxima, sums and outputs joined through LDS, sixteen
    // rows at a time: thread x then has four channels of row x / (D / 4)
    // and of every 256 / (D / 4)-th after it.
    constexpr int kLanes = D / 4, kStep = 256 / kLanes;
    const int my_ch = 4 * (threadIdx.x % kLanes);
    auto& wm = lds.m;
    auto& ws = lds.sum;
    auto& wo = lds.o;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (g4 == 0) {
            wm[wave][16 * nt + r16] = st[nt].m;
            ws[wave][16 * nt + r16] = st[nt].sum;
        }
#pragma unroll
        for (int x = 0; x < kUnit; ++x) {
            // Channels [g dim/4, ..) in order: unit 4 g + i, tile c.
            f32x4 v;
#pragma unroll
            for (int y = 0; y < 4; ++y) v[y] = o[nt][(4 * x + y) % kUnit][(4 * x + y) / kUnit];
            *reinterpret_cast<f32x4*>(&wo[wave][r16][(D / 4) * g4 + 4 * x]) = v;
        }
        __syncthreads();
#pragma unroll
        for (int r = threadIdx.x / kLanes; r < 16; r += kStep) {
            const int row = rt.begin + 16 * nt + r;
            if (row >= rt.end) break;
            float top = wm[0][16 * nt + r];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, wm[w][16 * nt + r]);
            const float keep = top == -__builtin_inff() ? 0.0f : top;
            float total = 0.0f;
            f32x4 acc{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(wm[w][16 * nt + r] - keep);
                total += f * ws[w][16 * nt + r];
                acc += f * *reinterpret_cast<const f32x4*>(&wo[w][r][my_ch]);
            }
            put(16 * nt + r, my_ch, acc, top, total);
        }
        if (nt + 1 < NT) __syncthreads();
    }
}

template <class E, int D, int kReach, int NT>
__global__ __launch_bounds__(256, (FewLds<D, NT>::kResident)) void kv_attention_kernel(AttendArgs a)
{
    constexpr int kRows = 16 * NT;
    __shared__ FewLds<D, NT> lds;
    const Batch& t = a.batch;
    const int h = blockIdx.x % t.kv_heads;
    const int split = blockIdx.x / t.kv_heads;
    Item it;
    if (!item_of(a, kRows, it)) return;
    const int b = it.b;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    const RowTile rt = row_tile<kReach>(a, it.index, kRows, len, n);
    if (rt.end <= rt.begin) return;
    const int tiles = tiles_of(a, rt);
    const int tile_begin = split * a.split_tiles;
    if (split > 0 && tile_begin >= tiles) return;
    const int tile_end = tile_begin + a.split_tiles < tiles ? tile_begin + a.split_tiles : tiles;
    const int active = (tiles + a.split_tiles - 1) / a.split_tiles;
    const int64_t item = it.id * t.kv_heads + h;
    const int64_t my_part = part_of(a, b, q0, h, split);
    few_rows<E, D, kReach, NT>(
        a, lds, Piece{b, h, len, q0, n, tile_begin, tile_end, -1, rt},
        [&](int r, int my_ch, f32x4 acc, float top, float total) {
            const int row = rt.begin + r;
            if (active <= 1) {
                finish<E>(a, t, q0, h, row, my_ch, acc, top, total);
                return;
            }
            const int64_t at = my_part + row;
            float* const to = a.part_o + at * D + my_ch;
            float* const pm = a.part_ml + 2 * at;
            if (a.arrived != nullptr) {
                put2(to, acc[0], acc[1]);
                put2(to + 2, acc[2], acc[3]);
                if (my_ch == 0) put2(pm, top, total);
            } else {
                *reinterpret_cast<f32x4*>(to) = acc;
                if (my_ch == 0) *reinterpret_cast<float2*>(pm) = float2{top, total};
            }
        });
    constexpr int kLanes = D / 4, kStep = 256 / kLanes;
    const int my_ch = 4 * (threadIdx.x % kLanes);
    if (active <= 1) return;
    if (a.arrived == nullptr) return;
    // The workgroup that arrives last joins the splits, in their order
    // whichever that is.  Every access to the partial results is an atomic
    // of the whole device (put2, get2: as compiled, stores and loads with sc1
    // set, which write through the XCD's cache and read past it), so their
    // completion is all that the count has to wait for.  A release fence of
    // the device is the same wait behind a write-back of the XCD's cache, for
    // plain stores that there are none of here; it took 5 us a call.
    __shared__ int last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t before =
            __hip_atomic_fetch_add(a.arrived + item, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = before + 1 == static_cast<uint32_t>(active);
        if (last) __hip_atomic_store(a.arrived + item, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    __shared__ float jm[kJoinSplits][kRows], js[kJoinSplits][kRows];
    const int64_t first_part = part_of(a, b, q0, h, 0) + rt.begin;
    for (int x = threadIdx.x; x < active * kRows; x += 256) {
        const int w = x / kRows, r = x % kRows;
        if (rt.begin + r >= rt.end) continue;
        const float2 v = get2(a.part_ml + 2 * (first_part + w * a.part_count + r));
        jm[w][r] = v.x;
        js[w][r] = v.y;
    }
    __syncthreads();
    for (int r = threadIdx.x / kLanes; rt.begin + r < rt.end; r += kStep) {
        float top = -__builtin_inff();
        for (int w = 0; w < active; ++w) top = fmaxf(top, jm[w][r]);
        const float keep = top == -__builtin_inff() ? 0.0f : top;
        float total = 0.0f;
        f32x4 acc{0, 0, 0, 0};
        const float* const po = a.part_o + (first_part + r) * D + my_ch;
#pragma unroll 4
        for (int w = 0; w < active; ++w) {
            const float f = __builtin_amdgcn_exp2f(jm[w][r] - keep);
            total += f * js[w][r];
            const float* const from = po + w * a.part_count * D;
            const float2 lo = get2(from), hi = get2(from + 2);
            acc += f * f32x4{lo.x, lo.y, hi.x, hi.y};
        }
        finish<E>(a, t, q0, h, rt.begin + r, my_ch, acc, top, total);
    }
}

// Rows of a workgroup of kv_attention_wide_kernel.
constexpr int kWideRows = 128;
constexpr int kXcds = 8;

// LDS of a workgroup of long chunks: a turn's tiles as elements, twice.  R waves
// have rows of their own; with two, two waves share each row's positions.
template <int D, int kReach>
struct WideLds {
    static constexpr int kPer = D == 256 && kReach == kOwn ? 1 : 2;  // tiles a turn
    static constexpr int kResident = D == 256 && kReach != kOwn ? 1 : 2;
    u32x4 keys[2][kPer][D / 16][64];
    u32x4 values[2][kPer][D / 32][2][64];
};

// Long chunks: four waves of 32 rows each read the same positions.
//
// A tile of 32 positions is D / 16 products S^T += K Q^T and D / 16 products
// O^T += V^T P^T, all v_mfma_f32_32x32x16: beside them the vector unit keeps
// working (three of its instructions in the time of 16 matrix cycles cost 8%
// more time; beside the 16 x 16 x 32 products, 20%).  The order of the
// contracted index is chosen so that a lane's scores are its weights: lane
// (r, g) = (lane % 32, lane / 32)
//   * gets the scores of query r against positions 16 u + 8 g + e, e < 8, for
//     u = 0 and 1, which are the slots of P^T that it feeds to product u;
//   * feeds, as row r of V^T, channels [r dim/32, (r+1) dim/32), one a tile.
// Converting a tile's codes in every wave would take more vector instructions
// than the softmax.  So each wave converts a quarter of the keys and values
// into LDS, in the order in which lanes feed them to the products (16 bytes a
// lane, no bank conflicts), and all four read them from there.  A turn takes
// two tiles (one at 256 channels): while they are multiplied the next two are
// converted and two more requested; one barrier a turn.
//
// 2,048 tokens of 32 heads over 16,390 positions, 516 GFLOP: 0.52 to 0.63 ms by
// the chip's clock, 990 to 820 TFLOP/s, 0.72 to 0.60 of what a large matrix
// product of the library reaches.  The chip's power may bound it, which no
// recorded clock shows: with 64 rows a wave, one workgroup a CU, 256 workgroups
// took more than twice as long as 128 of the same did on half of the CUs; and
// one or two tiles a turn, or scores formed a turn ahead of their softmax, end
// within 3% of each other.  Without LDS, each wave converting for itself (16 x
// 16 products): 0.69 ms where this took 0.63.  At 256 channels (1.44 ms) the
// output and the queries leave 29 registers too few, spilled.
template <class E, int D, int kReach>
__device__ __forceinline__ void wide_rows(const AttendArgs& a, WideLds<D, kReach>& lds, const Piece& piece)
{
    using V8 = typename E::V8;
    constexpr int kRows = 32;
    constexpr int kKeys = D / 16;     // fragments of a tile's keys
    constexpr int kMine = kKeys / 4;  // of them a wave's
    constexpr int kTiles = D / 32;    // tiles of O
    constexpr int kPer = WideLds<D, kReach>::kPer;
    auto& keys = lds.keys;
    auto& values = lds.values;
    const Batch& t = a.batch;
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int r32 = lane % 32, g2 = lane / 32;
    const int h = piece.h, b = piece.b, len = piece.len, q0 = piece.q0, n = piece.n;
    const RowTile& all = piece.rows;
    const int tile_begin = piece.begin, tile_end = piece.end;
    const int hi_pos = all.last_pos + 1;
    const int first_see = all.first_pos + 1;  // positions that every row of the workgroup sees
    // This wave's rows; at a chunk's end maybe none, and it only converts.
    const int begin = all.begin + wave * kRows;
    const int end = begin + kRows < all.end ? begin + kRows : all.end;

    // Fragment j of the keys is of wave j / kMine: channels 16 kMine w + 8 kMine
    // g + 8 i + e, so that a lane's share of a tile is one load.
    V8 q[kKeys];
    const int row = begin + r32;
    const bool in = row < end;
    const int token = (in ? row : all.begin) / a.group;
    const int head = h * a.group + (in ? row : all.begin) % a.group;
    // Positions that the row sees, or, of a draft's token, the row of its bits.
    const int limit = kReach == kDraft ? (in ? q0 + token : -1) : !in ? 0 : kReach == kCross ? len : len - n + token + 1;
    {
        const uint16_t* const p = a.q.p + (q0 + token) * a.q.token_stride + head * a.q.head_stride;
#pragma unroll
        for (int j = 0; j < kKeys; ++j)
            q[j] = __builtin_bit_cast(
                V8, load8(p + 16 * kMine * (j / kMine) + 8 * kMine * g2 + 8 * (j % kMine), a.q.wide));
    }
    f32x16 o[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
    Row st;
    bool far = false;

    // This wave's share of a tile as it is in the cache: the key of one
    // position a lane (row r of S^T is position 16 u + 8 g + 4 a + b for
    // r = 16 u + 8 a + 4 g + b), and the values of eight, of product `half`.
    uint32_t kr[kPer][kMine], ks[kPer], vr[kPer][D == 64 ? 4 : 8], vs[kPer][2];
    const int half = wave / 2;
    const uint32_t my_key = 16 * (r32 / 16) + 8 * (r32 / 4 % 2) + 4 * (r32 / 8 % 2) + r32 % 4;
    const int my_block = 2 * half + g2;  // of eight positions
    const uint32_t key_at = my_key * (D / 2) + 8 * kMine * wave + 4 * kMine * g2;
    const uint32_t key_scale_at = my_key * (D / 32) + (16 * kMine * wave + 8 * kMine * g2) / 32;
    const uint32_t value_at = (my_block * 16 + r32 / 2) * (D / 4);
    const uint32_t value_scale_at = (my_block * (D / 32) + r32 * D / 1024) * 8;
    const auto request = [&](int x, uint32_t at) {
        const uint64_t tile = at;
        const uint8_t* const kc = a.k_codes + tile * (16 * D) + key_at;
        if constexpr (kMine == 1) {
            kr[x][0] = *reinterpret_cast<const uint32_t*>(kc);
        } else if constexpr (kMine == 2) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(kc);
            kr[x][0] = v[0];
            kr[x][1] = v[1];
        } else {
            const u32x4 v = *reinterpret_cast<const u32x4*>(kc);
#pragma unroll
            for (int j = 0; j < 4; ++j) kr[x][j] = v[j];
        }
        ks[x] = (a.k_scales + tile * D)[key_scale_at];
        const uint8_t* const vp = a.v_codes + tile * (16 * D) + value_at;
        if constexpr (D == 256) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                vr[x][e] = *reinterpret_cast<const uint32_t*>(vp + 8 * e + 4 * (r32 % 2));
        } else {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(vp + 16 * c);
#pragma unroll
                for (int j = 0; j < 4; ++j) vr[x][4 * c + j] = v[j];
            }
        }
        const u32x2 s = *reinterpret_cast<const u32x2*>(a.v_scales + tile * D + value_scale_at);
        vs[x][0] = s[0];
        vs[x][1] = s[1];
    };
    // .. and as elements in LDS.  word: the tile's filter; the scale of a
    // position that no row sees, which may be anything, becomes 1.
    const auto convert = [&](auto kind, int x, int buf, uint32_t word) {
        const uint32_t sc = ks[x] << 23;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            keys[buf][x][wave * kMine + i][lane] =
                u32x4{E::template decode<0>(kr[x][i], sc), E::template decode<1>(kr[x][i], sc),
                      E::template decode<2>(kr[x][i], sc), E::template decode<3>(kr[x][i], sc)};
        if (D == 64 && wave % 2 != 0) return;  // one byte a position: two waves convert
        uint32_t scale[8];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            scale[4 * w] = vs[x][w] << 23;
            scale[4 * w + 1] = vs[x][w] << 15;
            scale[4 * w + 2] = vs[x][w] << 7;
            scale[4 * w + 3] = vs[x][w] >> 1;
        }
        if constexpr (decltype(kind)::value) {
            const uint32_t mine = word >> (16 * half + 8 * g2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!(mine >> e & 1u)) scale[e] = 127u << 23;
                if constexpr (kReach == kDraft) scale[e] = written_scale<E>(scale[e]);
            }
        }
        // Bytes of a lane's that this wave converts: D = 128: byte w % 2 of two,
        // D = 256: bytes 2 (w % 2) and that plus 1 of four.
        constexpr int kOwn = D == 256 ? 2 : 1;
#pragma unroll
        for (int y = 0; y < kOwn; ++y) {
            const int byte = D == 64 ? 0 : D == 128 ? wave % 2 : 2 * (wave % 2) + y;
            uint32_t g[2];  // the byte of four positions each
            if constexpr (D == 64) {
                const uint32_t pick = 0x06040200u + 0x01010101u * (r32 % 2);
                g[0] = __builtin_amdgcn_perm(vr[x][1], vr[x][0], pick);
                g[1] = __builtin_amdgcn_perm(vr[x][3], vr[x][2], pick);
            } else {
                const uint32_t at = D == 128 ? 2 * (r32 % 2) + byte : byte;
                const uint32_t low = 0x0C0C0400u + 0x0101u * at, high = 0x04000C0Cu + 0x01010000u * at;
                g[0] = __builtin_amdgcn_perm(vr[x][1], vr[x][0], low) | __builtin_amdgcn_perm(vr[x][3], vr[x][2], high);
                g[1] = __builtin_amdgcn_perm(vr[x][5], vr[x][4], low) | __builtin_amdgcn_perm(vr[x][7], vr[x][6], high);
            }
            const uint32_t d[8] = {
                E::template decode<0>(g[0], scale[0]), E::template decode<1>(g[0], scale[1]),
                E::template decode<2>(g[0], scale[2]), E::template decode<3>(g[0], scale[3]),
                E::template decode<0>(g[1], scale[4]), E::template decode<1>(g[1], scale[5]),
                E::template decode<2>(g[1], scale[6]), E::template decode<3>(g[1], scale[7])};
            u32x4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                even[j] = __builtin_amdgcn_perm(d[2 * j + 1], d[2 * j], 0x05040100u);
                odd[j] = __builtin_amdgcn_perm(d[2 * j + 1], d[2 * j], 0x07060302u);
            }
            values[buf][x][2 * byte][half][lane] = even;
            values[buf][x][2 * byte + 1][half][lane] = odd;
        }
    };
    // Fragments are read from LDS kAhead at a time, before their products.
    constexpr int kAhead = D == 128 ? 8 : 4;
    const auto multiply = [&](auto kind, int buf, const int (&from)[kPer], const uint32_t (&mine)[kPer]) {
        f32x16 s[kPer];
        [[maybe_unused]] Sees sees[kPer];
        if constexpr (decltype(kind)::value && kReach == kDraft) {
#pragma unroll
            for (int x = 0; x < kPer; ++x) {
                sees[x] = load_sees(a, limit, from[x] - (len - n));
            }
        }
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
#pragma unroll
            for (int lead = 0; lead < kKeys; lead += kAhead) {
                u32x4 f[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) f[j] = keys[buf][x][lead + j][lane];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    s[x] = E::mfma(__builtin_bit_cast(V8, f[j]), q[lead + j], s[x]);
            }
            if constexpr (decltype(kind)::value && kReach == kDraft) {
                const uint32_t ok = (mine[x] & sees_bits(sees[x], limit, from[x] - (len - n))) >> (8 * g2);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        s[x][8 * u + e] = (ok >> (16 * u + e) & 1u) ? s[x][8 * u + e] : -__builtin_inff();
            } else if constexpr (decltype(kind)::value) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    int left = limit - from[x] - 16 * u - 8 * g2;
                    left = left < 0 ? 0 : left > 8 ? 8 : left;
                    const uint32_t ok = mine[x] >> (16 * u + 8 * g2) & ((1u << left) - 1u);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        s[x][8 * u + e] = (ok >> e & 1u) ? s[x][8 * u + e] : -__builtin_inff();
                }
            }
        }
        // As weigh(), for 16 scores a tile and lane and two lanes a row.
        float top = s[0][0];
#pragma unroll
        for (int x = 0; x < kPer; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[x][i]);
        top *= a.scale_log2;
        if (far || __any(top - st.m > kSlack + E::kRaise)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            bool is_far;
            const float f = renew<E>(st, top, is_far);
#pragma unroll
            for (int c = 0; c < kTiles; ++c) o[c] *= f;
            far = __any(is_far);
            if (is_far) {
#pragma unroll
                for (int x = 0; x < kPer; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[x][i] = far_score(s[x][i], a.scale_log2, st.m);
            }
        }
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            V8 p[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][8 * u + e], a.scale_log2, -st.mu));
                    st.sum += w[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) p[u][e] = static_cast<typename E::T>(w[e]);
            }
#pragma unroll
            for (int lead = 0; lead < 2 * kTiles; lead += kAhead) {
                u32x4 f[kAhead];
#pragma unroll
                for (int y = 0; y < kAhead; ++y) f[y] = values[buf][x][(lead + y) / 2][y % 2][lane];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int y = u; y < kAhead; y += 2)
                        o[(lead + y) / 2] = E::mfma(__builtin_bit_cast(V8, f[y]), p[u], o[(lead + y) / 2]);
            }
        }
    };

    const int page_tiles_shift = t.page_shift - 5;
    for (int base = tile_begin; base < tile_end; base += 64) {
        int tile = base + lane;
        uint32_t at = 0, word = 0;
        int page = -1;
        if (tile < tile_end) {
            if (kReach != kOwn && a.live != nullptr) {
                const u32x4 entry = reinterpret_cast<const u32x4*>(a.live)[b * a.live_stride + tile];
                tile = entry[0];
                word = entry[1];
                page = entry[2];
            } else {
                page = t.page(b, tile >> page_tiles_shift);
                if (page >= 0) {
                    word = t.word(b, tile);
                    if (hi_pos - tile * kTile < 32) word &= (1u << (hi_pos - tile * kTile)) - 1u;
                }
            }
        }
        if (page >= 0)
            at = ((static_cast<uint32_t>(page) * t.kv_heads + h) << page_tiles_shift) +
                 (tile & ((1 << page_tiles_shift) - 1));
        else
            word = 0;
        const int t0 = tile * kTile;
        // The same in every wave: tiles that every row sees whole, kPer a turn,
        // then the others.
        uint64_t whole = __ballot(word == 0xFFFFFFFFu && t0 + kTile <= first_see);
        if (kPer == 2 && __popcll(whole) % 2 != 0) whole &= whole - 1;
        const uint64_t part = __ballot(word != 0) & ~whole;
        const auto run = [&](auto kind, uint64_t live) {
            if (live == 0) return;
            int i[kPer], next[kPer];
            uint32_t mine[kPer], ahead[kPer];
            // The next kPer tiles; past the last one it stands in, masked.
            const auto take = [&](int (&to)[kPer], uint32_t (&filter)[kPer], int last) {
#pragma unroll
                for (int x = 0; x < kPer; ++x) {
                    const bool some = live != 0;
                    to[x] = some ? __builtin_ctzll(live) : last;
                    live &= live - 1;
                    last = to[x];
                    filter[x] = some ? static_cast<uint32_t>(__builtin_amdgcn_readlane(word, to[x])) : 0u;
                    request(x, __builtin_amdgcn_readlane(at, to[x]));
                }
            };
            take(i, mine, 0);
#pragma unroll
            for (int x = 0; x < kPer; ++x) convert(kind, x, 0, mine[x]);
            bool more = live != 0;
            if (more) take(next, ahead, i[kPer - 1]);
            __syncthreads();
            int buf = 0;
            while (true) {
                int from[kPer];
                uint32_t now[kPer];
#pragma unroll
                for (int x = 0; x < kPer; ++x) {
                    from[x] = __builtin_amdgcn_readlane(t0, i[x]);
                    now[x] = mine[x];
                }
                const bool turn = more;
                if (turn) {
#pragma unroll
                    for (int x = 0; x < kPer; ++x) {
                        convert(kind, x, buf ^ 1, ahead[x]);
                        i[x] = next[x];
                        mine[x] = ahead[x];
                    }
                    more = live != 0;
                    if (more) take(next, ahead, i[kPer - 1]);
                }
                // Waves without rows, past a chunk's end, only convert.
                if (kReach == kOwn || begin < end) multiply(kind, buf, from, now);
                __syncthreads();
                if (!turn) break;
                buf ^= 1;
            }
        };
        run(std::false_type{}, whole);
        run(std::true_type{}, part);
    }

    st.sum += __shfl_xor(st.sum, 32);
    if (!in) return;
    if constexpr (kReach != kOwn) {
        if (piece.slot >= 0) {  // joined with the others by kv_join_pieces_kernel
            const int64_t to = static_cast<int64_t>(piece.slot) * kWideRows + wave * kRows + r32;
            if (g2 == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * to) = float2{st.m, st.sum};
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int z = 0; z < kTiles; ++z) {
                    f32x4 v;
#pragma unroll
                    for (int y = 0; y < 4; ++y) v[y] = o[(4 * z + y) % kTiles][4 * x + (4 * z + y) / kTiles];
                    *reinterpret_cast<f32x4*>(a.part_o + to * D + kTiles * (8 * x + 4 * g2) + 4 * z) = v;
                }
            return;
        }
    }
    uint16_t* const p = a.out.p + (q0 + token) * a.out.token_stride + head * a.out.head_stride;
    const float inv = st.sum != 0.0f ? 1.0f / st.sum : 0.0f;
    // Rows 8 x + 4 g + y of O^T, y < 4, hold channels dim/32 (8 x + 4 g) ..
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int z = 0; z < kTiles / 2; ++z) {
            u32x4 v;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int ch = 8 * z + 2 * y;
                typename E::V2 e;
                e[0] = static_cast<typename E::T>(o[ch % kTiles][4 * x + ch / kTiles] * inv);
                e[1] = static_cast<typename E::T>(o[(ch + 1) % kTiles][4 * x + ch / kTiles] * inv);
                v[y] = __builtin_bit_cast(uint32_t, e);
            }
            asm("" : "+v"(v));
            store8(p + kTiles * (8 * x + 4 * g2) + 8 * z, v, a.out.wide);
        }
    if (a.lse != nullptr && g2 == 0)
        a.lse[static_cast<int64_t>(q0 + token) * t.kv_heads * a.group + head] =
            (st.m + __builtin_log2f(st.sum)) * 0.69314718055994531f;
}

template <class E, int D>
__global__ __launch_bounds__(256, 2) void kv_attention_wide_kernel(AttendArgs a)
{
    __shared__ WideLds<D, kOwn> lds;
    const Batch& t = a.batch;
    Piece p;
    p.h = blockIdx.x;
    p.b = blockIdx.z;
    p.len = t.length(p.b);
    p.q0 = t.first_query(p.b);
    p.n = t.new_tokens(p.b, p.q0);
    const int index = gridDim.y - 1 - blockIdx.y;  // the longest rows first
    p.rows = row_tile<kOwn>(a, index, kWideRows, p.len, p.n);
    if (p.rows.end <= p.rows.begin) return;
    p.begin = 0;
    p.end = tiles_of(a, p.rows);
    p.slot = -1;
    wide_rows<E, D, kOwn>(a, lds, p);
}

// Tiles of a sequence of len positions that may have a page.
__device__ __forceinline__ int paged_tiles(const Batch& t, int len)
{
    const int last = len < t.max_positions ? len : t.max_positions;
    return (last + kTile - 1) / kTile;
}

// Tiles of a sequence that are looked at.
__device__ __forceinline__ int shared_tiles(const AttendArgs& a, int b, int len)
{
    return a.live != nullptr ? a.live_count[b] : paged_tiles(a.batch, len);
}

// What it takes to begin a row tile (its queries, the first tiles' way from
// memory, the part result), in tiles: they are counted into a workgroup's share.
// Beginning took 5 to 6 us, a tile of 128 channels 0.6 to 1.1; uncounted, a share
// of ten short sequences took 82 us where the others took 48.
constexpr int kStartTiles = 6;
// Of few rows, where four waves take a tile each: 32 drafts of 16 tokens on 500
// to 16,000 positions take 81 us with 6, 73 with 10, 67 with 16 and 24, 74 with 48.
constexpr int kStartFew = 16;

// More tiles than a call counts: the host takes other ways from here on.
constexpr int kMostCounted = (1 << 30) - 1;

// Row tiles of a sequence of n tokens, at most as many as there is room for.
__device__ __forceinline__ int shared_row_tiles(const AttendArgs& a, int rows, int n)
{
    const int64_t tiles = (static_cast<int64_t>(n) * a.group + rows - 1) / rows;
    return tiles < a.row_tiles ? static_cast<int>(tiles) : a.row_tiles;
}

// The same for drafts and cross attention, whose rows all reach the same
// positions, shared out evenly: the tiles of all sequences, key/value heads and
// row tiles stand in one line, and each workgroup takes as long a piece of it,
// whatever the sequences' lengths, which only the device knows.  A workgroup's
// piece may end one row tile, hold others whole and begin another: those that it
// holds in part (at most two) go to slots of their own, which
// kv_join_pieces_kernel joins.  Row tiles of one sequence and head stand next to
// each other and a piece goes to the XCD that has its neighbours, so that they
// find their positions in its L2.  32 drafts of 16 tokens, 32 heads to 8, on 500 to
// 16,000 positions under a filter (109 MB) take 65 to 69 us with the list and the
// join, 80 by splits of one length, whose 5,600 workgroups each had a beginning; 8
// of 63 tokens, 64 heads, on 4,000 to 30,000 (186 GFLOP) 232 to 250 us, 745 to 800
// TFLOP/s; 60 on 200,001 (393 GFLOP) 430 to 460, 855 to 915, within what the causal
// kernel reaches.
template <int kReach, int kRows, int kStart, class F>
__device__ __forceinline__ void share_out(const AttendArgs& a, F&& work)
{
    const Batch& t = a.batch;
    const int lane = threadIdx.x % 64;
    Piece p;
    p.b = 0;
    int s = 0, share = 1, from = 0, to = 1, index, padded = 0;
    if (a.split_tiles == 0) {  // so many row tiles that each is a workgroup's
        p.b = blockIdx.z;
        if (a.sequences <= 64) {
            // The longest sequences first, so that the last ones to run are short.
            const int mine = lane < a.sequences ? shared_tiles(a, lane, t.length(lane)) : -1;
            int before = 0;
            for (int b = 0; b < a.sequences; ++b) {
                const int other = __builtin_amdgcn_readlane(mine, b);
                before += other > mine || (other == mine && b < lane);
            }
            p.b = __builtin_ctzll(__ballot(before == p.b && lane < a.sequences));
        }
        p.h = blockIdx.x;
        index = blockIdx.y;
        p.begin = 0;
    } else {
        // Tiles of 64 sequences from b on, a sequence a lane: those of the lanes up
        // to this one, and this one's.  A sequence's own are below kMostCounted.
        const auto capped = [](int x) { return x < kMostCounted ? x : kMostCounted; };
        const auto tiles_from = [&](int b, int& own) {
            own = 0;
            if (b + lane < a.sequences) {
                const int len = t.length(b + lane), q0 = t.first_query(b + lane);
                own = shared_row_tiles(a, kRows, t.new_tokens(b + lane, q0)) *
                      (shared_tiles(a, b + lane, len) + kStart) * t.kv_heads;
            }
            int upto = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int x = __shfl_up(upto, d);
                if (lane >= d) upto = capped(upto + x);
            }
            return upto;
        };
        int total = 0, own, upto;
        for (int b = 0; b < a.sequences; b += 64) {
            upto = tiles_from(b, own);
            total = capped(total + __builtin_amdgcn_readlane(upto, 63));
        }
        if (total == 0) return;
        if (total == kMostCounted) {
            // Row offsets that overlap give more than the host bounds: no row tile
            // is worked on, and all are noted as written.
            const int64_t all = static_cast<int64_t>(a.slots) * t.kv_heads;
            for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256)
                reinterpret_cast<int2*>(a.pieces)[i] = int2{-1, 0};
            return;
        }
        const int workgroups = gridDim.x;
        share = (total + workgroups - 1) / workgroups;
        if (share < a.split_tiles) share = a.split_tiles;
        share += share % 2;
        if (a.sequences == 1) {
            // All row tiles have as many tiles: parts that end with them.
            const int all = shared_tiles(a, 0, t.length(0));
            const int items = total / (all + kStart), room = workgroups / items;
            if (room > 0 && all > 0) {
                int parts = (all + share - 1) / share;
                parts = parts < room ? parts : room;
                share = (all + parts - 1) / parts;
                share += share % 2;
                parts = (all + share - 1) / share;
                padded = parts * share;
                total = items * padded;
            }
        }
        const int shares = (total + share - 1) / share;
        const int each = (shares + kXcds - 1) / kXcds;
        s = blockIdx.x % kXcds * each + blockIdx.x / kXcds;
        if (static_cast<int>(blockIdx.x / kXcds) >= each || s >= shares) return;
        from = s * share;
        to = from + share < total ? from + share : total;

        // Where the share begins.
        p.begin = from;
        if (padded == 0) {
            for (;; p.b += 64) {
                if (a.sequences > 64) upto = tiles_from(p.b, own);
                const int here = __builtin_amdgcn_readlane(upto, 63);
                if (p.begin < here) break;
                p.begin -= here;
            }
            const int at = __builtin_ctzll(__ballot(upto > p.begin));
            p.begin -= __builtin_amdgcn_readlane(upto - own, at);
            p.b += at;
        }
    }
    const int start = padded != 0 ? 0 : kStart;
    int count, tiles, row_tiles;  // the sequence's: tiles looked at, counted, row tiles
    const auto enter = [&] {
        p.len = t.length(p.b);
        p.q0 = t.first_query(p.b);
        p.n = t.new_tokens(p.b, p.q0);
        count = shared_tiles(a, p.b, p.len);
        tiles = padded != 0 ? padded : count + start;
        row_tiles = shared_row_tiles(a, kRows, p.n);
    };
    enter();
    if (a.split_tiles == 0) {
        if (index >= row_tiles) return;
        to = tiles;
    } else {
        const int unit = p.begin / tiles;
        p.begin -= unit * tiles;
        p.h = unit / row_tiles;
        index = unit - p.h * row_tiles;
    }
    for (int at = from; at < to;) {
        const int left = to - at;
        const int counted = p.begin, counted_end = left < tiles - counted ? counted + left : tiles;
        p.begin = counted > start ? counted - start : 0;
        p.end = counted_end > start ? counted_end - start : 0;
        if (p.end > count) p.end = count;
        // A row tile with nothing to read is written by the share that begins it.
        if (p.begin < p.end || (count == 0 && counted == 0)) {
            p.rows = row_tile<kReach>(a, index, kRows, p.len, p.n);
            p.slot = p.begin == 0 && p.end == count ? -1 : 2 * s + (at != from);
            if (p.begin == 0 && a.split_tiles != 0 && threadIdx.x == 0) {
                // The row tile's first slot, and how many shares after it have a part.
                const int64_t id = (a.slots == 0 ? static_cast<int64_t>(p.b) * a.row_tiles
                                                 : static_cast<int64_t>(p.q0) * a.group / kRows + p.b) + index;
                reinterpret_cast<int2*>(a.pieces)[id * t.kv_heads + p.h] =
                    int2{p.slot, (at - counted + tiles - 1) / share - s};
            }
            work(p);
        }
        at += counted_end - counted;
        p.begin = 0;
        if (++index < row_tiles) continue;
        index = 0;
        if (++p.h < t.kv_heads) continue;
        p.h = 0;
        if (at >= to) break;
        do {
            ++p.b;
            enter();
        } while (p.n == 0);
    }
}

// .. by 128 rows a workgroup,
template <class E, int D, int kReach>
__global__ __launch_bounds__(256, (WideLds<D, kReach>::kResident)) void kv_attention_shared_kernel(AttendArgs a)
{
    __shared__ WideLds<D, kReach> lds;
    share_out<kReach, kWideRows, kStartTiles>(a, [&](const Piece& p) { wide_rows<E, D, kReach>(a, lds, p); });
}

// .. and by few rows.
template <class E, int D, int kReach, int NT>
__global__ __launch_bounds__(256, (FewLds<D, NT>::kResident)) void kv_attention_shared_few_kernel(AttendArgs a)
{
    constexpr int kRows = 16 * NT;
    __shared__ FewLds<D, NT> lds;
    share_out<kReach, kRows, kStartFew>(a, [&](const Piece& p) {
        few_rows<E, D, kReach, NT>(a, lds, p, [&](int r, int ch, f32x4 acc, float top, float total) {
            if (p.slot < 0) {
                finish<E>(a, a.batch, p.q0, p.h, p.rows.begin + r, ch, acc, top, total);
                return;
            }
            const int64_t at = static_cast<int64_t>(p.slot) * kRows + r;
            *reinterpret_cast<f32x4*>(a.part_o + at * D + ch) = acc;
            if (ch == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = float2{top, total};
        });
        __syncthreads();  // LDS is free again
    });
}

// Joins the pieces of a row tile that several workgroups had a part of, D / 4
// lanes a row and 1 << a.join_shift such groups of lanes, each with its part of
// the pieces.  A lane looks up every D / 4-th piece's reference and sum, so that
// all are under way at once.
template <class E, int D, int kReach, int kRows>
__global__ __launch_bounds__(256) void kv_join_pieces_kernel(AttendArgs a)
{
    constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
    __shared__ float2 stats[kGroups];
    __shared__ f32x4 theirs[kGroups][kLanes];
    const Batch& t = a.batch;
    const int h = blockIdx.x % t.kv_heads;
    const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    const int ways = 1 << a.join_shift, way = group & (ways - 1);
    const int r = (blockIdx.x / t.kv_heads * kGroups + group) >> a.join_shift;
    Item it;
    if (!item_of(a, kRows, it)) return;
    // Tokens beyond the host's bound: no share had them, and nothing was noted of them.
    if (it.index >= a.row_tiles) return;
    const int2 entry = reinterpret_cast<const int2*>(a.pieces)[it.id * t.kv_heads + h];
    const int len = t.length(it.b);
    const int q0 = t.first_query(it.b);
    const int n = t.new_tokens(it.b, q0);
    const RowTile rt = row_tile<kReach>(a, it.index, kRows, len, n);
    const int slot = entry.x, pieces = entry.y + 1;
    if (rt.end <= rt.begin || slot < 0) return;  // no such tile, or written already
    const bool in = rt.begin + r < rt.end;
    // The parts after the first begin their shares: slots 2 (slot / 2 + i).
    const auto row_of = [&](int i) {
        return static_cast<int64_t>(i == 0 ? slot : 2 * (slot / 2 + i)) * kRows + r;
    };
    float top = -__builtin_inff(), total = 0.0f;
    f32x4 acc{0, 0, 0, 0};
    for (int base = way; in && base < pieces; base += kLanes * ways) {
        float2 ml{-__builtin_inff(), 0.0f};
        if (base + lane * ways < pieces)
            ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * row_of(base + lane * ways));
        float fresh = ml.x;
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) fresh = fmaxf(fresh, __shfl_xor(fresh, d));
        fresh = fmaxf(fresh, top);
        const float keep = fresh == -__builtin_inff() ? 0.0f : fresh;
        const float old = __builtin_amdgcn_exp2f(top - keep);
        top = fresh;
        const float f = __builtin_amdgcn_exp2f(ml.x - keep);
        total = total * old + f * ml.y;  // a lane's own pieces
        acc *= old;
        int count = (pieces - base + ways - 1) >> a.join_shift;
        count = count < kLanes ? count : kLanes;
        // Loads in batches, past the last one again that one: a loop of single ones
        // for what a batch leaves would wait for each.
        constexpr int kBatch = 4;
        for (int i = 0; i < count; i += kBatch) {
            f32x4 x[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int at = i + k < count ? i + k : count - 1;
                x[k] = *reinterpret_cast<const f32x4*>(a.part_o + row_of(base + at * ways) * D + 4 * lane);
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const float w = __shfl(f, (i + k) & (kLanes - 1), kLanes);
                if (i + k < count) acc += w * x[k];
            }
        }
    }
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) total += __shfl_xor(total, d);
    if (ways > 1) {
        if (lane == 0) stats[group] = float2{top, total};
        theirs[group][lane] = acc;
        __syncthreads();
        if (way != 0) return;
        for (int w = 1; w < ways; ++w) top = fmaxf(top, stats[group + w].x);
        const float keep = top == -__builtin_inff() ? 0.0f : top;
        total = 0.0f;
        acc = f32x4{0, 0, 0, 0};
        for (int w = 0; w < ways; ++w) {
            const float f = __builtin_amdgcn_exp2f(stats[group + w].x - keep);
            total += f * stats[group + w].y;
            acc += f * theirs[group + w][lane];
        }
    }
    if (in) finish<E>(a, t, q0, h, rt.begin + r, 4 * lane, acc, top, total);
}

// Joins the splits' partial results of one row: four waves a row, wave w the
// splits w, w + 4, .., each lane D / 64 channels.
template <class E, int D, int kReach, int NT>
__global__ __launch_bounds__(256) void kv_join_kernel(AttendArgs a)
{
    constexpr int kRows = 16 * NT;
    constexpr int kC = D / 64;
    __shared__ float wo[4][D], wm[4], ws[4];
    const Batch& t = a.batch;
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int h = blockIdx.x % t.kv_heads;
    const int r = blockIdx.x / t.kv_heads;
    Item it;
    if (!item_of(a, kRows, it)) return;
    const int index = it.index, b = it.b;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    const RowTile rt = row_tile<kReach>(a, index, kRows, len, n);
    const int row = rt.begin + r;
    if (row >= rt.end) return;
    const int active = (tiles_of(a, rt) + a.split_tiles - 1) / a.split_tiles;
    if (active <= 1) return;  // written already
    const int64_t at = part_of(a, b, q0, h, 0) + row;
    const float* const ml = a.part_ml + 2 * at;
    const float* const po = a.part_o + at * D + lane * kC;
    float top = -__builtin_inff(), total = 0.0f;
    float acc[kC] = {};
    for (int base = wave; base < active; base += 256) {
        // Lane l has split base + 4 l.
        const int s = base + 4 * lane;
        const float m = s < active ? ml[2 * s * a.part_count] : -__builtin_inff();
        const float z = s < active ? ml[2 * s * a.part_count + 1] : 0.0f;
        float fresh = m;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) fresh = fmaxf(fresh, __shfl_xor(fresh, d));
        fresh = fmaxf(fresh, top);
        const float keep = fresh == -__builtin_inff() ? 0.0f : fresh;
        const float old = __builtin_amdgcn_exp2f(top - keep);
        top = fresh;
        const float f = __builtin_amdgcn_exp2f(m - keep);
        total = total * old + f * z;  // a lane's own splits
#pragma unroll
        for (int c = 0; c < kC; ++c) acc[c] *= old;
        int count = (active - base + 3) / 4;
        count = count < 64 ? count : 64;
        for (int k = 0; k < count; ++k) {
            const float fk = __builtin_bit_cast(
                float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), k));
#pragma unroll
            for (int c = 0; c < kC; ++c)
                acc[c] += fk * po[(base + 4 * k) * a.part_count * D + c];
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
#pragma unroll
    for (int c = 0; c < kC; ++c) wo[wave][lane * kC + c] = acc[c];
    if (lane == 0) {
        wm[wave] = top;
        ws[wave] = total;
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) >= D) return;
    const float all = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    const float keep = all == -__builtin_inff() ? 0.0f : all;
    float sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(wm[w] - keep);
        sum += f * ws[w];
        o += f * wo[w][threadIdx.x];
    }
    const int i_tok = row / a.group, head = h * a.group + row % a.group;
    uint16_t* const p = a.out.p + (q0 + i_tok) * a.out.token_stride + head * a.out.head_stride;
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    p[threadIdx.x] = __builtin_bit_cast(uint16_t, static_cast<typename E::T>(o * inv));
    if (a.lse != nullptr && threadIdx.x == 0)
        a.lse[static_cast<int64_t>(q0 + i_tok) * t.kv_heads * a.group + head] =
            (all + __builtin_log2f(sum)) * 0.69314718055994531f;
}

// How a call is cut up, chosen on the host.
struct AttendPlan {
    int nt;      // 16-row tiles a wave holds
    bool wide;   // four row tiles a workgroup over the same positions
    bool shared; // drafts, cross attention: few rows, their tiles shared out
    dim3 grid, join;
};

// One launch each; defined per element type, dim and reach.
template <class E, int D, int kReach>
void attend_launch(const AttendArgs& a, const AttendPlan& p, hipStream_t stream)
{
    if constexpr (kReach == kOwn) {
        if (p.wide) {
            kv_attention_wide_kernel<E, D><<<p.grid, 256, 0, stream>>>(a);
            return;
        }
    } else {
        if (p.wide) {
            kv_attention_shared_kernel<E, D, kReach><<<p.grid, 256, 0, stream>>>(a);
            if (a.split_tiles != 0) kv_join_pieces_kernel<E, D, kReach, kWideRows><<<p.join, 256, 0, stream>>>(a);
            return;
        }
        if (p.shared) {
            const auto few = [&](auto nt) {
                constexpr int kNt = decltype(nt)::value;
                kv_attention_shared_few_kernel<E, D, kReach, kNt><<<p.grid, 256, 0, stream>>>(a);
                kv_join_pieces_kernel<E, D, kReach, 16 * kNt><<<p.join, 256, 0, stream>>>(a);
            };
            if constexpr (D == 256) {
                if (p.nt == 1) return few(std::integral_constant<int, 1>{});
            }
            return few(std::integral_constant<int, 2>{});
        }
    }
    const auto run = [&](auto nt) {
        constexpr int kNt = decltype(nt)::value;
        kv_attention_kernel<E, D, kReach, kNt><<<p.grid, 256, 0, stream>>>(a);
        if (a.splits > 1 && a.arrived == nullptr)
            kv_join_kernel<E, D, kReach, kNt><<<p.join, 256, 0, stream>>>(a);
    };
    if constexpr (D < 256) {
        if (p.nt == 2) return run(std::integral_constant<int, 2>{});
    }
    run(std::integral_constant<int, 1>{});
}

// The instantiations: one file for each dim and reach.
#define GOFANN_KV_ATTEND(kind, D, reach)                                                       \
    kind template void attend_launch<Bf16, D, reach>(const AttendArgs&, const AttendPlan&,     \
                                                     hipStream_t);                             \
    kind template void attend_launch<F16, D, reach>(const AttendArgs&, const AttendPlan&,      \
                                                    hipStream_t)
#define GOFANN_KV_ATTEND_EXTERN(reach)   \
    GOFANN_KV_ATTEND(extern, 64, reach); \
    GOFANN_KV_ATTEND(extern, 128, reach); \
    GOFANN_KV_ATTEND(extern, 256, reach)
GOFANN_KV_ATTEND_EXTERN(kOwn);
GOFANN_KV_ATTEND_EXTERN(kDraft);
GOFANN_KV_ATTEND_EXTERN(kCross);

}  // namespace kv
}  // namespace gofann
