// kv_cache.hip -- host side of the attention over the 4-bit key/value cache:
// how a call is cut into row tiles and splits, and its launches.
#include "kv_attention.hpp"

namespace gofann {
namespace kv {
namespace {

// The tiles of a sequence that its filter leaves something of, in order: tile,
// filter word and page, a place of four words each.  A workgroup lists 1,024
// tiles and counts for itself what lies before them.
constexpr int kLiveChunk = 1024;
__global__ __launch_bounds__(256) void kv_live_kernel(AttendArgs a, u32x4* live, int32_t* count)
{
    __shared__ int part[4];
    const Batch& t = a.batch;
    const int b = blockIdx.y;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int len = t.length(b);
    const int tiles = paged_tiles(t, len);
    const int begin = blockIdx.x * kLiveChunk;
    if (begin > 0 && begin >= tiles) return;
    const auto word_of = [&](int tile) -> uint32_t {
        if (tile >= tiles) return 0u;
        const int left = (len < t.max_positions ? len : t.max_positions) - tile * kTile;
        return t.word(b, tile) & (left < kTile ? (1u << left) - 1u : 0xFFFFFFFFu);
    };
    int before = 0;
#pragma unroll 8
    for (int tile = threadIdx.x; tile < begin; tile += 256) before += word_of(tile) != 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) before += __shfl_xor(before, d);
    if (lane == 0) part[wave] = before;
    __syncthreads();
    before = part[0] + part[1] + part[2] + part[3];
    __syncthreads();
    // Four tiles a thread, next to each other.
    uint32_t word[4];
    int own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        word[i] = word_of(begin + 4 * threadIdx.x + i);
        own += word[i] != 0;
    }
    int upto = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int x = __shfl_up(upto, d);
        if (lane >= d) upto += x;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int at = before + upto - own;
    for (int w = 0; w < wave; ++w) at += part[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (word[i] == 0) continue;
        const int tile = begin + 4 * threadIdx.x + i;
        const int page = t.page(b, tile >> (t.page_shift - 5));
        live[static_cast<int64_t>(b) * a.live_stride + at++] =
            u32x4{static_cast<uint32_t>(tile), word[i], static_cast<uint32_t>(page), 0};
    }
    if (begin + kLiveChunk >= tiles && threadIdx.x == 255) count[b] = at;
}

}  // namespace
}  // namespace kv

namespace {

// Rows up to which a sequence of a long-chunk launch is left to the other kernel.
constexpr int kFewRows = 64;

// Bytes of partial results that a call may have; past them splits get longer.
// They are a million rows of a split (128 channels), at most 32 to a workgroup,
// so that the chip is full all the same.
constexpr uint64_t kPartBytes = 512ull << 20;

// Tiles of a split of `items` row tiles of at most `most` tiles: three workgroups
// a CU (two to five are resident, by the kernel), at least one tile a wave,
// and where sequences may differ in length at most 48, so that a long one does
// not outlast the others: 48 sequences of 500 to 16,000 positions take 64 us
// with 16, 55 with 32, 52 with 48 and 56 with 64; 8 of them 19, 21, 18 and 18.
int split_tiles(const Context* ctx, uint64_t items, uint64_t most, bool ragged, uint64_t max_splits)
{
    const uint64_t resident = 3ull * static_cast<uint64_t>(ctx->compute_units);
    uint64_t n = (items * most + resident - 1) / resident;
    n = (n + 3) / 4 * 4;
    if (n < 4) n = 4;
    // Few enough for the last workgroup to join, where that costs a wave at
    // most two tiles: 64 listed blocks of 64 positions, eight heads, take 9.0 us
    // in 16 splits and 12 in 32 with a launch of the join.
    const uint64_t few = (most + kv::kJoinSplits - 1) / kv::kJoinSplits;
    if (n < few && few <= 8) n = few;
    if (ragged && n > 48) n = 48;
    const uint64_t least = (most + max_splits - 1) / max_splits;
    if (n < least) n = (least + 3) / 4 * 4;
    return static_cast<int>(n);
}

// Sequences whose tiles a workgroup counts for itself, 64 at a time.  Past it
// nothing is lost: 1,100 of 16 tokens, 32 heads to 8, on 100 to 2,000 positions take
// 620 us by splits, 730 shared out; of 80 tokens 2,720 and 3,430.
constexpr uint32_t kMostShared = 1024;

// Whether drafts and cross attention of `rows` rows a sequence share their tiles
// out by 128 rows a workgroup, not by 16 or 32: past 256, where their row tiles
// are nearly as full.  8 sequences of 2,000 to 16,000 positions, eight key/value
// heads, us by few / by 128 rows: 128 channels: 128 rows 42 / 47, 256 rows 81 / 89,
// 384 rows 123 / 117; 64 channels: 59 / 59 and 87 / 76 of 256 and 384; 19 drafts of
// 280 rows of 64 channels 27 / 33.  One sequence of 2,800 rows, which goes by 128, would
// be faster by few: of 128 channels on 3,055 positions 63 / 70, of 64 on 6,502 77 / 83.
//
// 256 channels, four heads: 384, 1,024 and 2,000 rows of 16 sequences of 1,000 to 4,000
// positions 111 / 115, 292 / 279 and 538 / 480; of 8 of 2,000 to 16,000 161 / 168,
// 387 / 403 and 673 / 700; of 2 of 10,000 65 / 80, 140 / 160 and 219 / 244.  They go by
// 128 rows for the first; the others lose 4 to 22% by it.  One sequence stays with few
// rows further: 1,024 rows on 40,000 positions 239 / 284, on 10,000 76 / 97.
//
// The longest sequence decides for all.  One of 700 tokens among 63 of one token on 700
// to 8,000 positions, 32 heads to 8, which goes by 128 rows: 64 channels 137 / 177, 128
// 125 / 201, 256 411 / 783; a single token's row tile is as long as a full one's.
bool many_rows(uint64_t rows, uint32_t dim, uint32_t sequences)
{
    return rows > (dim == 256 && sequences == 1 ? 2048u : 256u) &&
           10 * ((rows + 127) / 128 * 128) <= 11 * ((rows + 31) / 32 * 32);
}

// Tiles of 16 rows a wave that has few of them.  Two have no room for a second
// wave a SIMD at 256 channels and pay there where there is much to read: 128 rows
// on 40,000 positions 78 us, 90 with one; on 4,000 24.7 and 24.2; 72 rows on 40,000
// 66 and 65.5.
uint64_t few_tiles(uint64_t rows, uint32_t dim, uint64_t most_tiles)
{
    if (rows <= 16) return 1;
    return dim < 256 || (rows >= 128 && most_tiles > 256) ? 2 : 1;
}

// Whether few rows share their tiles out at all: up to 16 rows, whose kernels
// have no registers left for it, and short calls, which a second launch would
// lengthen, keep splits of one length, joined by the last of them.  64 rows of 128
// channels, eight key/value heads, us by splits / shared out: 16 sequences of 250 to
// 1,000 positions 17.9 / 21.5, four of 2,000 18.2 / 20.0, four of 1,000 to 4,000
// 21.6 / 21.5, 16 of 500 to 2,000 25.1 / 25.8, 16 of 1,000 to 16,000 58 / 48, 32 of 500
// to 16,000 under a filter 80 / 63.  One of 1,000 13.8 / 14.3, of 2,100 20.2 / 14.4; from
// some 1,200 to 2,048 a single one, which stays with splits, loses by it: of 1,500
// 17.0 / 14.4, of 2,000 18.8 / 14.6 (64 channels 14.3 / 12.4, 256 23.6 / 15.5).
bool share_few(uint64_t rows, uint32_t dim, uint64_t items, uint64_t most_tiles, int compute_units)
{
    return rows > 16 && (most_tiles > 64 || items * most_tiles * dim >= 4096ull * compute_units);
}

// Tiles of a share at least, us with 8 / 16 / 32.  64 rows of 128 channels: one
// sequence of 2,500 positions 14.5 / 15.7 / 17.7, of 8,000 18.8 / 16.4 / 18.8; four of
// 2,500 21.0 / 21.6 / 21.5, of 4,000 23.8 / 23.7 / 25.5; with more the shares are
// longer anyway.  512 rows, by 128: one sequence of 2,100 26.1 / 25.0 / 29.3, of 4,000
// 30.7 / 29.1 / 36.1; four of 1,000 to 2,000 41.2 / 41.7 / 42.3.
int least_share(bool wide, uint32_t sequences) { return wide || sequences == 1 ? 8 : 16; }

// Bytes that the list of the tiles that a filter leaves may have.
constexpr uint64_t kLiveBytes = 64ull << 20;

// How the tiles of drafts or of cross attention are shared out.
struct AttendShape {
    uint64_t row_tiles;   // of a sequence at most
    uint64_t slots;       // as AttendArgs has it
    uint64_t counted;     // tiles that the device counts, at most
    uint32_t workgroups;  // shares; 0: every row tile is a workgroup's
    int join_shift;
    dim3 where;           // row tiles
    uint64_t o_bytes, ml_bytes, piece_bytes, live_bytes, count_bytes;
    uint64_t bytes() const { return o_bytes + ml_bytes + piece_bytes + live_bytes + count_bytes; }
};

AttendShape shared_shape(const Context* ctx, const gofann_kv_cache* cache, const gofann_kv_batch* batch,
                         uint64_t group, uint64_t tokens, uint64_t most_tiles, uint64_t per)
{
    using namespace kv;
    AttendShape s{};
    const uint64_t heads = cache->kv_heads;
    s.row_tiles = (tokens * group + per - 1) / per;
    uint64_t all = s.row_tiles * batch->sequences;
    const uint64_t slots = batch->queries * group / per + batch->sequences;
    const dim3 grid(static_cast<uint32_t>(heads), static_cast<uint32_t>(s.row_tiles), batch->sequences);
    s.where = grid;
    if (batch->query_offsets != nullptr && 2 * slots <= all && slots <= 0x7FFFFFFFu) {
        s.slots = all = slots;
        s.where.y = slots < 65535 ? static_cast<uint32_t>(slots) : 65535u;
        s.where.z = static_cast<uint32_t>((slots + s.where.y - 1) / s.where.y);
    }
    s.counted = (all + s.row_tiles) * heads * (most_tiles + kStartFew);
    // Workgroups that are resident: two a CU; of 128 or 32 rows of 256 channels one
    // (LDS, registers).  A third of 32 rows of 64 channels gave 1% on average.
    const bool wide = per == kWideRows;
    const uint64_t each = cache->dim == 256 && per > 16 ? 1 : 2;
    uint64_t workgroups = each * static_cast<uint64_t>(ctx->compute_units) / kXcds * kXcds;
    if (workgroups == 0) workgroups = kXcds;
    const uint64_t items = (batch->queries * group + per - 1) / per * heads;
    // Enough row tiles to even out by themselves, the longest first, save the
    // parts' way through memory: 6 x 701 tokens on 900 to 7,000 positions take 233
    // us, 245 shared out; 4,096 on 5,000 345 and 364.  Not at 256 channels: 8 x 500
    // tokens on 8,000 take 866, and 697 shared out.
    // Nor are those of a call counted that may have too many tiles for it.
    if (wide && (s.counted >= kMostCounted || (s.slots == 0 && cache->dim < 256 && 2 * items >= 3 * workgroups))) {
        s.slots = 0;
        s.where = grid;
        return s;
    }
    s.workgroups = static_cast<uint32_t>(workgroups);
    // Row tiles in so many parts that a lane group has about eight of them.
    const int most_shift = cache->dim == 256 ? 2 : 3;  // four lane groups a workgroup
    while (s.join_shift < most_shift && (8ull << s.join_shift) * items < workgroups) ++s.join_shift;
    const uint64_t parts = 2 * workgroups * per;
    s.o_bytes = parts * cache->dim * sizeof(float);
    s.ml_bytes = parts * 2 * sizeof(float);
    s.piece_bytes = (all * heads * 2 * sizeof(int32_t) + 15) / 16 * 16;
    // Where a filter may hide whole tiles, those that are left are listed and
    // shared out: 16 drafts of 64 tokens on 1,000 to 16,000 positions, 0.6 of them
    // visible in documents of 40 to 700, take 104 us, 121 without the list.
    const uint64_t live = batch->visible == nullptr ? 0 : batch->sequences * most_tiles * 4 * sizeof(uint32_t);
    if (live <= kLiveBytes) {
        s.live_bytes = live;
        s.count_bytes = live > 0 ? batch->sequences * sizeof(int32_t) : 0;
    }
    return s;
}

}  // namespace

int kv_attention(Context* ctx, const gofann_kv_cache* cache, const gofann_kv_batch* batch,
                 const gofann_kv_rows* q, uint32_t heads, float scale, const int32_t* blocks,
                 uint32_t width, const gofann_kv_rows* out, float* out_lse, const KvReach& reach)
{
    using namespace kv;
    AttendArgs a{};
    a.sees = reach.sees;
    a.sees_stride = static_cast<int64_t>(reach.sees_stride);
    a.sees_width = static_cast<int>(reach.sees_width);
    a.batch = batch_of(cache, batch);
    a.q = rows_of(q);
    a.out = rows_of(out);
    a.k_codes = cache->k_codes;
    a.k_scales = cache->k_scales;
    a.v_codes = cache->v_codes;
    a.v_scales = cache->v_scales;
    a.blocks = blocks;
    a.lse = out_lse;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.group = static_cast<int>(heads / cache->kv_heads);
    a.width = static_cast<int>(width);
    const uint32_t dim = cache->dim;
    const uint32_t tokens = batch->query_offsets == nullptr ? 1 : batch->max_queries;
    const uint32_t most_tiles =
        blocks != nullptr ? width * (cache->page_size / kTile)
                          : (static_cast<uint32_t>(a.batch.max_positions) + kTile - 1) / kTile;
    const auto launch = [&](const AttendArgs& x, const AttendPlan& p) {
        const auto of_reach = [&](auto kind) {
            constexpr int kReach = decltype(kind)::value;
            const bool bf = cache->elem == GOFANN_ELEM_BF16;
            switch (dim) {
                case 64: (bf ? attend_launch<Bf16, 64, kReach> : attend_launch<F16, 64, kReach>)(x, p, ctx->stream); break;
                case 128: (bf ? attend_launch<Bf16, 128, kReach> : attend_launch<F16, 128, kReach>)(x, p, ctx->stream); break;
                default: (bf ? attend_launch<Bf16, 256, kReach> : attend_launch<F16, 256, kReach>)(x, p, ctx->stream); break;
            }
        };
        if (reach.cross)
            of_reach(std::integral_constant<int, kCross>{});
        else if (reach.sees != nullptr)
            of_reach(std::integral_constant<int, kDraft>{});
        else
            of_reach(std::integral_constant<int, kOwn>{});
    };
    const bool own = !reach.cross && reach.sees == nullptr;
    const auto fail = [&](int code, const char* what) {
        const char* const call = own ? "kv_attention: " : reach.cross ? "kv_cross_attention: " : "kv_draft_attention: ";
        return ctx->fail(code, std::string(call) + what);
    };
    const char* const too_many = "too many tokens a sequence for one call";
    uint64_t rows = blocks != nullptr ? static_cast<uint64_t>(a.group)
                                      : static_cast<uint64_t>(tokens) * a.group;
    a.rows_upto = 0x7FFFFFFF;
    a.sequences = static_cast<int>(batch->sequences);
    uint64_t part_rows = static_cast<uint64_t>(batch->queries) * a.group;

    // Long chunks, where they fill the chip: by the rows that there are, not by
    // sequences times the longest.  Sequences of few rows among them, such as
    // the decoding ones of a mixed batch, would each keep a workgroup busy with
    // all of their positions; they are left to the other kernel.
    const uint64_t all_rows = static_cast<uint64_t>(batch->queries) * a.group;
    if (own && blocks == nullptr && rows > kFewRows &&
        all_rows / kWideRows * cache->kv_heads >= static_cast<uint64_t>(ctx->compute_units)) {
        AttendPlan p{};
        p.wide = true;
        const uint64_t row_tiles = (rows + kWideRows - 1) / kWideRows;
        if (row_tiles > 65535) return fail(GOFANN_ERR_UNSUPPORTED, too_many);
        a.splits = 1;
        a.split_tiles = static_cast<int>(most_tiles);
        a.row_tiles = static_cast<int>(row_tiles);
        const bool mixed = static_cast<uint64_t>(batch->sequences) * tokens > batch->queries;
        a.rows_over = mixed ? kFewRows : 0;
        p.grid = dim3(cache->kv_heads, static_cast<uint32_t>(row_tiles), batch->sequences);
        launch(a, p);
        if (hipGetLastError() != hipSuccess) return fail(GOFANN_ERR_HIP, "launch");
        if (!mixed) return GOFANN_OK;
        a.rows_over = 0;
        a.rows_upto = kFewRows;
        rows = kFewRows;
        if (static_cast<uint64_t>(batch->sequences) * kFewRows < part_rows) {
            a.part_rows = kFewRows;
            part_rows = static_cast<uint64_t>(batch->sequences) * kFewRows;
        }
    }

    // Drafts and cross attention: tiles shared out.
    const bool many = many_rows(rows, dim, batch->sequences);
    const uint64_t per_few = 16 * few_tiles(rows, dim, most_tiles);
    const uint64_t few_items = (all_rows + per_few - 1) / per_few * cache->kv_heads;
    if (!own && blocks == nullptr && batch->sequences <= kMostShared &&
        (many || share_few(rows, dim, few_items, most_tiles, ctx->compute_units))) {
        AttendPlan p{};
        p.wide = many;
        p.shared = !many;
        p.nt = static_cast<int>(per_few / 16);
        const uint64_t per = many ? kWideRows : per_few;
        const AttendShape shape = shared_shape(ctx, cache, batch, a.group, tokens, most_tiles, per);
        if (shape.row_tiles > 65535) return fail(GOFANN_ERR_UNSUPPORTED, too_many);
        // Tiles are counted in 32 bits.  Few rows that may have too many go by splits:
        // 1,024 sequences of 64 rows, eight heads, from 2,100,000 positions on.
        if (shape.workgroups == 0 || shape.counted < kMostCounted) {
            a.row_tiles = static_cast<int>(shape.row_tiles);
            a.slots = static_cast<int>(shape.slots);
            if (shape.workgroups == 0) {
                p.grid = shape.where;
            } else {
                a.split_tiles = least_share(many, batch->sequences);
                a.join_shift = shape.join_shift;
                a.live_stride = most_tiles;
                char* const w = static_cast<char*>(ctx->workspace(Context::kScratchKv, shape.bytes()));
                if (w == nullptr) return GOFANN_ERR_NOMEM;
                a.part_o = reinterpret_cast<float*>(w);
                a.part_ml = reinterpret_cast<float*>(w + shape.o_bytes);
                a.pieces = reinterpret_cast<int32_t*>(w + shape.o_bytes + shape.ml_bytes);
                if (shape.live_bytes > 0) {
                    char* const live = w + shape.o_bytes + shape.ml_bytes + shape.piece_bytes;
                    char* const count = live + shape.live_bytes;
                    a.live = reinterpret_cast<uint32_t*>(live);
                    a.live_count = reinterpret_cast<int32_t*>(count);
                    kv_live_kernel<<<dim3((most_tiles + kLiveChunk - 1) / kLiveChunk, batch->sequences), 256, 0,
                                     ctx->stream>>>(a, reinterpret_cast<u32x4*>(live),
                                                    reinterpret_cast<int32_t*>(count));
                }
                p.grid = dim3(shape.workgroups);
                const uint32_t lanes = static_cast<uint32_t>(per) * dim / 4 << shape.join_shift;
                p.join = dim3(cache->kv_heads * lanes / 256, shape.where.y, shape.where.z);
            }
            launch(a, p);
            if (hipGetLastError() != hipSuccess) return fail(GOFANN_ERR_HIP, "launch");
            return GOFANN_OK;
        }
    }

    // Two 16-row tiles a wave past 16 rows: 32 rows of 128 channels over 8 x
    // 30,000 positions, two heads, take 31.6 us, and 48 rows 39.  At 256
    // channels they do not fit the registers: 119 us with spills, 65 as two
    // tiles of 16.
    AttendPlan p{};
    p.nt = rows <= 16 || dim == 256 ? 1 : 2;
    const uint32_t per = 16 * p.nt;
    a.token_tiles = static_cast<int>((a.group + per - 1) / per);
    const uint64_t row_tiles =
        blocks != nullptr ? static_cast<uint64_t>(tokens) * a.token_tiles : (rows + per - 1) / per;
    if (row_tiles > 65535) return fail(GOFANN_ERR_UNSUPPORTED, too_many);
    a.row_tiles = static_cast<int>(row_tiles);
    // Tiles counted through the sequences where a grid of them is twice as many:
    // 63 sequences of one token and one of 128, 32 heads to 8, up to 8,192
    // positions, take 87 us so and 138 by the grid.  Where it is not, splits are
    // sized for tiles that are not there: 19 sequences of five tokens take 36, and
    // 25 by the grid.
    uint64_t all_tiles = row_tiles * batch->sequences;
    dim3 where(0, static_cast<uint32_t>(row_tiles), batch->sequences);
    const uint64_t slots = blocks != nullptr
                               ? static_cast<uint64_t>(batch->queries) * a.token_tiles
                               : static_cast<uint64_t>(batch->queries) * a.group / per + batch->sequences;
    if (batch->query_offsets != nullptr && 2 * slots <= all_tiles && slots <= 0x7FFFFFFFu) {
        a.slots = static_cast<int>(slots);
        all_tiles = slots;
        where.y = slots < 65535 ? static_cast<uint32_t>(slots) : 65535u;
        where.z = static_cast<uint32_t>((slots + where.y - 1) / where.y);
    }
    const uint64_t items = all_tiles * cache->kv_heads;
    const uint64_t a_split = part_rows * cache->kv_heads * (dim + 2) * sizeof(float);
    const uint64_t max_splits = a_split < kPartBytes ? kPartBytes / a_split : 1;
    a.split_tiles = split_tiles(ctx, items, most_tiles, batch->sequences > 1, max_splits);
    a.splits = most_tiles > 0 ? static_cast<int>((most_tiles + a.split_tiles - 1) / a.split_tiles) : 1;
    if (a.splits > 1) {
        const uint64_t parts = part_rows * cache->kv_heads * static_cast<uint64_t>(a.splits);
        const size_t o_bytes = parts * dim * sizeof(float);
        char* const w = static_cast<char*>(
            ctx->workspace(Context::kScratchKv, o_bytes + parts * 2 * sizeof(float)));
        if (w == nullptr) return GOFANN_ERR_NOMEM;
        if (a.splits <= kJoinSplits) {
            a.arrived = static_cast<uint32_t*>(ctx->zeroed(Context::kScratchKvArrived, items * 4));
            if (a.arrived == nullptr) return GOFANN_ERR_NOMEM;
        }
        a.part_count = static_cast<int64_t>(part_rows);
        a.part_o = reinterpret_cast<float*>(w);
        a.part_ml = reinterpret_cast<float*>(w + o_bytes);
    }
    p.grid = dim3(cache->kv_heads * static_cast<uint32_t>(a.splits), where.y, where.z);
    p.join = dim3(cache->kv_heads * per, where.y, where.z);
    launch(a, p);
    if (hipGetLastError() != hipSuccess) return fail(GOFANN_ERR_HIP, "launch");
    return GOFANN_OK;
}

}  // namespace gofann
