// kv_select.hip -- the blocks of the paged 4-bit key/value cache that each
// token and key/value head reads: integer scores of the queries against the
// pages' boxes, then the highest `width` of them in ascending order.
#include "device_common.hpp"
#include "kv_common.hpp"

namespace gofann {
namespace kv {
namespace {

constexpr int kChunk = 256;                   // blocks that a workgroup scores: 16 tiles of 16
constexpr int kRepeat = 4;                    // token tiles that a workgroup scores in turn
constexpr int kBins = 2048;
constexpr uint32_t kForced = 0xFFFFFFFFu;     // above every score's key
constexpr uint32_t kIneligible = 0;           // below every score's key

struct SelectArgs {
    Batch batch;
    Rows q;
    const int8_t* box;
    const uint8_t* box_scale;
    uint32_t* keys;     // [queries][kv_heads][key_stride], where a row has several chunks
    int64_t key_stride;
    uint32_t* arrived;  // [item], zero between calls: chunks scored; NULL: kv_pick_kernel picks
    int32_t* out;
    int group;        // heads a key/value head
    int group_shift;  // log2 of the rows a token's heads take of a 16-row tile
    int tokens;       // tokens of a tile, a power of two
    int token_tiles;  // tiles of a sequence
    int head_tiles;   // 16-row tiles of one token's heads, where they are more than 16
    int width, first, last;
};

// Position of token i of sequence b, and the blocks up to it; none below 0.
__device__ __forceinline__ int position(int len, int n, int i) { return len - n + i; }

__device__ __forceinline__ int blocks_to(const Batch& t, int pos)
{
    return pos < 0 ? 0 : (pos >> t.page_shift) + 1;
}

// Those of `blocks` that may have a page.
__device__ __forceinline__ int paged(const Batch& t, int blocks)
{
    const int most = (t.max_positions + (1 << t.page_shift) - 1) >> t.page_shift;
    return blocks < most ? blocks : most;
}

// Whether block j (page_size positions) has a visible position up to pos.
__device__ __forceinline__ bool any_visible(const Batch& t, int b, int j, int pos)
{
    if (t.visible == nullptr) return true;
    if (pos >= t.max_positions) pos = t.max_positions - 1;
    const int words = 1 << (t.page_shift - 5);
    const int w0 = j * words;
    uint32_t any = 0;
    for (int w = w0; w < w0 + words && 32 * w <= pos; ++w) {
        const int left = pos + 1 - 32 * w;
        const uint32_t cut = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
        any |= t.word(b, w) & cut;
    }
    return any != 0;
}

// Keys pass between workgroups of one launch as accesses of device scope.
__device__ __forceinline__ void put(uint32_t* p, uint32_t x)
{
    __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t get(const uint32_t* p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x)
{
    const auto shifted = [](uint32_t v, auto ctrl, auto rows) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
            0, static_cast<int>(v), decltype(ctrl)::value, decltype(rows)::value, 0xF, true));
    };
    using std::integral_constant;
    x += shifted(x, integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr 1
    x += shifted(x, integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
    x += shifted(x, integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
    x += shifted(x, integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
    x += shifted(x, integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // lane 15 on
    x += shifted(x, integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // lane 31 on
    return x;
}

struct PickShared {
    __attribute__((aligned(16))) uint32_t hist[kBins];
    uint32_t part[4][4];
    uint32_t found[3];
};

// The `width` highest of a row's keys, their blocks written in ascending
// order.  The range of the keys is cut into 2048 bins, the bin that the last
// taken key falls into becomes the range, until the number wanted of it is all
// of it or one key is left, of which the lowest blocks are taken: two rounds
// for keys that differ, at most three.  Wave w has the w-th quarter of the
// blocks, N keys a lane in registers where they all fit.  load(j): the j-th key.
template <int N, class L>
__device__ void pick(const SelectArgs& a, PickShared& sh, int blocks, int32_t* out, L&& load)
{
    const int tid = threadIdx.x, lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int span = (blocks + 255) / 256 * 64;
    const int begin = wave * span;
    const int end = begin + span < blocks ? begin + span : blocks;
    const bool held = span <= 64 * N;
    uint32_t k[N];
    const auto fetch = [&](int from) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = from + 64 * i + lane;
            k[i] = j < end ? load(j) : kIneligible;
        }
    };
    // f(key, block) for every block of the wave, all lanes together.
    const auto visit = [&](auto&& f) {
        if (held) {
#pragma unroll
            for (int i = 0; i < N; ++i) f(k[i], begin + 64 * i + lane);
        } else {
            for (int from = begin; from < end; from += 64 * N) {
                fetch(from);
#pragma unroll
                for (int i = 0; i < N; ++i) f(k[i], from + 64 * i + lane);
            }
        }
    };
    if (held) fetch(begin);

    uint32_t forced = 0, open = 0, least = 0xFFFFFFFFu, most = 0;
    visit([&](uint32_t key, int) {
        const bool is_open = key != kForced && key != kIneligible;
        forced += __popcll(__ballot(key == kForced));
        open += __popcll(__ballot(is_open));
        const uint32_t l = is_open ? key : 0xFFFFFFFFu, m = is_open ? key : 0u;
        least = l < least ? l : least;
        most = m > most ? m : most;
    });
    least = wave_min_u32(least);
    most = wave_max_u32(most);
#pragma unroll
    for (int x = tid; x < kBins / 4; x += 256) reinterpret_cast<u32x4*>(sh.hist)[x] = u32x4{0, 0, 0, 0};
    if (lane == 0) *reinterpret_cast<u32x4*>(sh.part[wave]) = u32x4{forced, open, least, most};
    __syncthreads();
    forced = open = most = 0;
    least = 0xFFFFFFFFu;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(sh.part[w]);
        forced += v[0];
        open += v[1];
        least = v[2] < least ? v[2] : least;
        most = v[3] > most ? v[3] : most;
    }
    uint32_t want = static_cast<uint32_t>(a.width) - forced;
    // Taken: keys above `limit`, and the first `want` that equal it.
    uint32_t limit;
    if (open <= want) {
        limit = 0;
        want = 0;
    } else if (want == 0) {
        limit = kForced - 1;
    } else {
        while (true) {
            limit = least;
            if (least == most) break;
            const int bits = 32 - __builtin_clz(most - least);
            const int shift = bits > 11 ? bits - 11 : 0;
            visit([&](uint32_t key, int) {
                if (key >= least && key <= most) atomicAdd(&sh.hist[(key - least) >> shift], 1u);
            });
            __syncthreads();
            // Thread x has eight bins, the highest first; they are cleared for
            // the next round as they are read.
            constexpr int kOwn = kBins / 256;
            const int low = kBins - kOwn * (tid + 1);
            uint32_t c[kOwn], sum = 0;
#pragma unroll
            for (int m = 0; m < kOwn; m += 4) {
                u32x4* const at = reinterpret_cast<u32x4*>(sh.hist + low + m);
                const u32x4 v = *at;
                *at = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    c[m + y] = v[y];
                    sum += v[y];
                }
            }
            uint32_t upto = wave_scan(sum);
            if (lane == 63) sh.part[wave][0] = upto;
            __syncthreads();
            for (int w = 0; w < wave; ++w) upto += sh.part[w][0];
            uint32_t above = upto - sum;
            if (above < want && upto >= want) {
#pragma unroll
                for (int m = kOwn - 1; m >= 0; --m) {
                    if (above < want && above + c[m] >= want) {
                        sh.found[0] = static_cast<uint32_t>(low + m);
                        sh.found[1] = above;
                        sh.found[2] = c[m];
                    }
                    above += c[m];
                }
            }
            __syncthreads();
            want -= sh.found[1];
            least += sh.found[0] << shift;
            if (sh.found[2] == want) {  // all of the bin
                limit = least - 1;
                want = 0;
                break;
            }
            const uint32_t last = least + ((1u << shift) - 1u);
            most = last < most ? last : most;
        }
    }
    // Every wave writes behind what the waves before it take.
    uint32_t above = 0, equal = 0;
    visit([&](uint32_t key, int) {
        above += __popcll(__ballot(key > limit));
        equal += __popcll(__ballot(key == limit && key != kIneligible));
    });
    __syncthreads();
    if (lane == 0) *reinterpret_cast<u32x2*>(sh.part[wave]) = u32x2{above, equal};
    __syncthreads();
    uint32_t at = 0, seen = 0, total = 0, ties = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(sh.part[w]);
        if (w < wave) {
            at += v[0];
            seen += v[1];
        }
        total += v[0];
        ties += v[1];
    }
    total += ties < want ? ties : want;
    at += seen < want ? seen : want;
    const uint64_t below = (1ull << lane) - 1ull;
    visit([&](uint32_t key, int j) {
        const bool is_tie = key == limit && key != kIneligible;
        const uint64_t eq = __ballot(is_tie);
        const uint64_t take = __ballot(key > limit || (is_tie && seen + __popcll(eq & below) < want));
        if (take >> lane & 1ull) out[at + __popcll(take & below)] = j;
        at += __popcll(take);
        seen += __popcll(eq);
    });
    for (uint32_t j = total + tid; j < static_cast<uint32_t>(a.width); j += 256) out[j] = -1;
}

// The same from the keys that the scores left in memory.
__device__ void pick_row(const SelectArgs& a, PickShared& sh, int blocks, int64_t row)
{
    const uint32_t* const keys = a.keys + row * a.key_stride;
    if (blocks <= 2048)
        pick<8>(a, sh, blocks, a.out + row * a.width, [&](int j) { return get(keys + j); });
    else
        pick<16>(a, sh, blocks, a.out + row * a.width, [&](int j) { return get(keys + j); });
}

// Scores of 256 blocks for a tile of tokens, or several: one token a sequence
// is picked for by the last workgroup to finish, more by a launch of their own,
// a workgroup each, so that a workgroup here may score one tile of tokens after
// the other against the same boxes (2 x 300 tokens, 4 heads, up to 625 blocks:
// 50 us with the last workgroup picking for two tokens in turn, 33 so).  The rows of an i8 product are a token's heads (each token
// padded to a power of two of rows by repeating its last head, which changes
// no maximum), the columns blocks: a lane then holds four heads of one block,
// and the maximum over a token's heads stays in the lane and its neighbours
// 16 and 32 lanes away.  sum_c max(q most, q least) is one product of length
// 2 dim, of the positive part of q with `most` and the negative with `least`.
//
// 16 sequences of 20,000 to 131,000 positions, 8 heads (38 MB of boxes): 18.4
// us, 2.1 TB/s.  One long row after the other, latency bounds it: of 12.5 us for
// one sequence 7.8 are the chain from its length over pages and queries to
// the boxes and keys, 0.5 the count of arrivals, 4.2 the choice.
// kQuads: a token has at least four rows, so a lane's four are one token's.
// kMany: more than one token a sequence.
template <class E, int D, bool kQuads, bool kMany>
__global__ __launch_bounds__(256, D == 256 ? 2 : 3) void kv_select_kernel(SelectArgs a)
{
    constexpr int K = D / 64;               // products of 64 channels
    constexpr int kBatch = D == 256 ? 2 : 4;  // 16-block tiles requested at once
    __shared__ uint32_t stage[kChunk];  // the keys, where one chunk is all
    __shared__ PickShared sh;
    __shared__ int is_last;
    const Batch& t = a.batch;
    const int h = blockIdx.x % t.kv_heads;
    const int chunk = blockIdx.x / t.kv_heads;
    const int b = blockIdx.z;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int r16 = lane % 16, g4 = lane / 16;
    // Pages are looked up beside the sequence's length, which may rule them out.
    int early[kBatch];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) early[x] = t.page(b, chunk * kChunk + 16 * (wave + 4 * x) + r16);
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    const int rows_shift = a.group_shift;  // rows a token takes: 1 << rows_shift
    const int per = kMany ? a.tokens * kRepeat : 1;
    const int first_token = kMany ? blockIdx.y * per : 0;
    if (first_token >= n) return;
    const int stop = first_token + per < n ? first_token + per : n;
    const int blocks = paged(t, blocks_to(t, position(len, n, stop - 1)));
    const int chunks = (blocks + kChunk - 1) / kChunk;
    if (chunk > 0 && chunk >= chunks) return;
    const bool whole = !kMany && chunks <= 1;  // all keys of the row are here

    // Positive and negative part of the quantized queries, 16 channels a lane
    // and product; the rows' powers of two.
    i32x4 qp[K], qn[K];
    int unit[4];
    uint32_t raw[K][8];
    const auto request_queries = [&](int i0, int ht) {
        int i = i0 + (r16 >> rows_shift);
        i = i < stop ? i : stop - 1;
        int head = 16 * ht + (r16 & ((1 << rows_shift) - 1));
        head = head < a.group ? head : a.group - 1;
        const uint16_t* const row = a.q.p + (q0 + i) * a.q.token_stride +
                                    (static_cast<int64_t>(h) * a.group + head) * a.q.head_stride;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const u32x4 v = load8(row + 64 * k + 16 * g4 + 8 * half, a.q.wide);
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[k][4 * half + j] = v[j];
            }
    };
    const auto quantize_queries = [&]() {
        // Magnitudes compare as the integers of their bits, two to a word.
        constexpr uint32_t kInf = std::is_same_v<E, Bf16> ? 0x7F80u : 0x7C00u;
        using U2 = uint16_t __attribute__((ext_vector_type(2)));
        const auto largest = [&]() {
            U2 m = {0, 0};
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    m = __builtin_elementwise_max(m, __builtin_bit_cast(U2, raw[k][j] & 0x7FFF7FFFu));
            uint32_t top = m[0] > m[1] ? m[0] : m[1];
            uint32_t other = __shfl_xor(top, 16);
            top = other > top ? other : top;
            other = __shfl_xor(top, 32);
            return other > top ? other : top;
        };
        uint32_t top = largest();
        if (__any(top >= kInf)) {
            // Infinities stay out of the maximum and saturate, a NaN is zero.
            uint32_t kept[K][8];
            for (int k = 0; k < K; ++k)
                for (int j = 0; j < 8; ++j) {
                    uint32_t w = raw[k][j], fin = w;
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t m = w >> (16 * half) & 0x7FFFu, mask = 0xFFFFu << (16 * half);
                        if (m > kInf) w &= ~mask;
                        if (m >= kInf) fin &= ~mask;
                    }
                    kept[k][j] = w;
                    raw[k][j] = fin;
                }
            top = largest();
            for (int k = 0; k < K; ++k)
                for (int j = 0; j < 8; ++j) raw[k][j] = kept[k][j];
        }
        const float amax = static_cast<float>(__builtin_bit_cast(typename E::V2, top)[0]);
        int e = amax > 0.0f ? __builtin_amdgcn_frexp_expf(amax) - 7 : -125;
        e = e < -125 ? -125 : e > 125 ? 125 : e;
        const float inv = __builtin_bit_cast(float, static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float f = static_cast<float>(
                        __builtin_bit_cast(typename E::V2, raw[k][2 * w + j / 2])[j % 2]);
                    // Rounded to nearest even in the low bits of a number of
                    // ulp 1; clamping to a whole number may come before it.
                    f = __builtin_amdgcn_fmed3f(f * inv, -127.0f, 127.0f) + 12582912.0f;
                    v[j] = __builtin_bit_cast(uint32_t, f);
                }
                const uint32_t x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], 0x0C0C0400u),
                                                         __builtin_amdgcn_perm(v[1], v[0], 0x0C0C0400u),
                                                         0x05040100u);
                const uint32_t sign = x >> 7 & 0x01010101u;
                const uint32_t mask = (sign << 8) - sign;  // 255 in every negative byte
                qp[k][w] = static_cast<int>(x & ~mask);
                qn[k][w] = static_cast<int>(x & mask);
            }
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) unit[i4] = __shfl(e, 4 * g4 + i4);
    };

    const int64_t row0 = static_cast<int64_t>(q0) * t.kv_heads + h;  // row of token i: + i kv_heads
    // Tiles of the chunk: wave w has w, w + 4, w + 8, w + 12.
    for (int batch = 0; batch < 4 / kBatch; ++batch) {
        int page[kBatch];
        int eb[kBatch];
        i32x4 hi[kBatch][K], lo[kBatch][K];
#pragma unroll
        for (int x = 0; x < kBatch; ++x) {
            const int block = chunk * kChunk + 16 * (wave + 4 * (batch * kBatch + x)) + r16;
            page[x] = batch == 0 ? early[x] : t.page(b, block);
            if (block >= blocks) page[x] = -1;
        }
        // The queries are requested between the pages and the boxes, so that
        // they are quantized while the boxes are on their way.
        if (batch == 0) request_queries(first_token, 0);
#pragma unroll
        for (int x = 0; x < kBatch; ++x) {
            const int64_t ph = static_cast<int64_t>(page[x] < 0 ? 0 : page[x]) * t.kv_heads + h;
            const int8_t* const p = a.box + ph * 2 * D + 16 * g4;
            const bool in = page[x] >= 0;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                hi[x][k] = in ? *reinterpret_cast<const i32x4*>(p + 64 * k) : i32x4{0, 0, 0, 0};
                lo[x][k] = in ? *reinterpret_cast<const i32x4*>(p + D + 64 * k) : i32x4{0, 0, 0, 0};
            }
            eb[x] = in ? static_cast<int>(a.box_scale[ph]) - 127 : 0;
        }
        for (int i0 = first_token; i0 < stop; i0 += kMany ? a.tokens : 1) {
            const int i_end = !kMany || i0 + a.tokens > stop ? stop : i0 + a.tokens;
            float s[kBatch][4];
            for (int ht = 0; ht < a.head_tiles; ++ht) {
                const bool others = kMany || a.head_tiles > 1;  // than the queries held
                if (ht > 0 || i0 > first_token || (batch > 0 && others)) request_queries(i0, ht);
                if (batch == 0 || others) quantize_queries();
#pragma unroll
                for (int x = 0; x < kBatch; ++x) {
                    i32x4 acc = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qp[k], hi[x][k], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qn[k], lo[x][k], acc, 0, 0, 0);
                    }
                    // |acc| < 2^23, so the conversion is exact, and so is the
                    // product wherever the result is a normal number: both
                    // powers at once, as one alone may leave the range.
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float f = __builtin_ldexpf(static_cast<float>(acc[i]), unit[i] + eb[x]);
                        s[x][i] = ht == 0 ? f : fmaxf(s[x][i], f);
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                // Maximum over a token's rows.
                const int block = chunk * kChunk + 16 * (wave + 4 * (batch * kBatch + x)) + r16;
                const auto write = [&](int first_row, float score) {
                    const int token = i0 + (first_row >> rows_shift);
                    if (token >= i_end) return;
                    const int pos = position(len, n, token);
                    const int upto = blocks_to(t, pos), mine = paged(t, upto);
                    uint32_t key = kIneligible;
                    if (block < mine && page[x] >= 0 && any_visible(t, b, block, pos)) {
                        const uint32_t u = __builtin_bit_cast(uint32_t, score + 0.0f);  // -0 as 0
                        key = (u & 0x80000000u) ? ~u : u | 0x80000000u;
                        if (block < a.first || block >= upto - a.last) key = kForced;
                    }
                    if (whole)
                        stage[block] = key;
                    else if (block < mine)
                        put(a.keys + (row0 + static_cast<int64_t>(token) * t.kv_heads) * a.key_stride + block,
                            key);
                };
                if constexpr (kQuads) {
                    float m = fmaxf(fmaxf(s[x][0], s[x][1]), fmaxf(s[x][2], s[x][3]));
                    if (rows_shift >= 3) m = fmaxf(m, __shfl_xor(m, 16));
                    if (rows_shift >= 4) m = fmaxf(m, __shfl_xor(m, 32));
                    if ((4 * g4 & ((1 << rows_shift) - 1)) == 0) write(4 * g4, m);
                } else if (rows_shift == 1) {
                    write(4 * g4, fmaxf(s[x][0], s[x][1]));
                    write(4 * g4 + 2, fmaxf(s[x][2], s[x][3]));
                } else {
                    for (int i = 0; i < 4; ++i) write(4 * g4 + i, s[x][i]);
                }
            }
        }
    }
    if constexpr (kMany) return;
    if (chunks > 1) {
        // The keys are atomics of the whole device (as compiled, stores and
        // loads with sc1 set, which no XCD's cache holds back), so that their
        // completion is all that the count has to wait for.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t* const count =
                a.arrived + (static_cast<int64_t>(b) * a.token_tiles + blockIdx.y) * t.kv_heads + h;
            const uint32_t before =
                __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            is_last = before + 1 == static_cast<uint32_t>(chunks);
            if (is_last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!is_last) return;
    } else {
        __syncthreads();
    }
    const int mine = paged(t, blocks_to(t, position(len, n, 0)));
    if (whole)
        pick<1>(a, sh, mine, a.out + row0 * a.width, [&](int j) { return stage[j]; });
    else
        pick_row(a, sh, mine, row0);
}

// One token and key/value head a workgroup.
__global__ __launch_bounds__(256) void kv_pick_kernel(SelectArgs a)
{
    __shared__ PickShared sh;
    const Batch& t = a.batch;
    const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    if (i >= n) return;
    pick_row(a, sh, paged(t, blocks_to(t, position(len, n, i))),
             static_cast<int64_t>(q0 + i) * t.kv_heads + h);
}

template <class E>
void launch(const SelectArgs& a, uint32_t dim, bool many, dim3 grid, hipStream_t stream)
{
    const auto run = [&](auto quads, auto many) {
        constexpr bool kQuads = decltype(quads)::value, kMany = decltype(many)::value;
        switch (dim) {
            case 64: kv_select_kernel<E, 64, kQuads, kMany><<<grid, 256, 0, stream>>>(a); break;
            case 128: kv_select_kernel<E, 128, kQuads, kMany><<<grid, 256, 0, stream>>>(a); break;
            default: kv_select_kernel<E, 256, kQuads, kMany><<<grid, 256, 0, stream>>>(a); break;
        }
    };
    if (a.group_shift >= 2)
        many ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});
    else
        many ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});
}

}  // namespace
}  // namespace kv

int kv_select(Context* ctx, const gofann_kv_cache* cache, const gofann_kv_batch* batch,
              const gofann_kv_rows* q, uint32_t heads, uint32_t width, uint32_t first,
              uint32_t last, int32_t* out_blocks)
{
    using namespace kv;
    SelectArgs a{};
    a.batch = batch_of(cache, batch);
    a.q = rows_of(q);
    a.box = cache->box;
    a.box_scale = cache->box_scale;
    a.out = out_blocks;
    a.group = static_cast<int>(heads / cache->kv_heads);
    while ((1 << a.group_shift) < a.group && a.group_shift < 4) ++a.group_shift;
    a.head_tiles = (a.group + 15) / 16;
    // At most four tokens a tile and its own picks.
    a.tokens = 16 >> a.group_shift;
    if (a.tokens > 4) a.tokens = 4;
    a.width = static_cast<int>(width);
    a.first = static_cast<int>(first);
    a.last = static_cast<int>(last);
    const uint32_t tokens = batch->query_offsets == nullptr ? 1 : batch->max_queries;
    if (tokens > 65535)
        return ctx->fail(GOFANN_ERR_UNSUPPORTED, "kv_select: at most 65535 tokens a sequence");
    const uint32_t per = tokens > 1 ? static_cast<uint32_t>(a.tokens * kRepeat) : 1u;
    a.token_tiles = static_cast<int>((tokens + per - 1) / per);
    const uint32_t most = static_cast<uint32_t>(a.batch.max_positions);
    const uint32_t blocks = (most + cache->page_size - 1) / cache->page_size;
    const uint32_t chunks = blocks > 0 ? (blocks + kChunk - 1) / kChunk : 1;
    if (chunks > 1 || tokens > 1) {
        a.key_stride = blocks;
        a.keys = static_cast<uint32_t*>(
            ctx->workspace(Context::kScratchKv,
                           static_cast<size_t>(batch->queries) * cache->kv_heads * (blocks + 1) * 4));
        if (a.keys == nullptr) return GOFANN_ERR_NOMEM;
    }
    if (chunks > 1 && tokens == 1) {
        a.arrived = static_cast<uint32_t*>(
            ctx->zeroed(Context::kScratchKvArrived,
                        static_cast<size_t>(batch->sequences) * cache->kv_heads * 4));
        if (a.arrived == nullptr) return GOFANN_ERR_NOMEM;
    }
    const dim3 grid(chunks * cache->kv_heads, static_cast<uint32_t>(a.token_tiles), batch->sequences);
    if (cache->elem == GOFANN_ELEM_BF16)
        launch<Bf16>(a, cache->dim, tokens > 1, grid, ctx->stream);
    else
        launch<F16>(a, cache->dim, tokens > 1, grid, ctx->stream);
    if (tokens > 1)
        kv_pick_kernel<<<dim3(cache->kv_heads, tokens, batch->sequences), 256, 0, ctx->stream>>>(a);
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_select: launch");
    return GOFANN_OK;
}

}  // namespace gofann
