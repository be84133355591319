// kv_cache.hip -- host side of the attention over the 4-bit key/value cache:
// how a call is cut into row tiles and splits, and its launches.
#include "kv_attention.hpp"

namespace gofann {
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

}  // namespace

int kv_attention(Context* ctx, const gofann_kv_cache* cache, const gofann_kv_batch* batch,
                 const gofann_kv_rows* q, uint32_t heads, float scale, const int32_t* blocks,
                 uint32_t width, const gofann_kv_rows* out, float* out_lse)
{
    using namespace kv;
    AttendArgs a{};
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
        const bool bf = cache->elem == GOFANN_ELEM_BF16;
        switch (dim) {
            case 64: (bf ? attend_launch<Bf16, 64> : attend_launch<F16, 64>)(x, p, ctx->stream); break;
            case 128: (bf ? attend_launch<Bf16, 128> : attend_launch<F16, 128>)(x, p, ctx->stream); break;
            default: (bf ? attend_launch<Bf16, 256> : attend_launch<F16, 256>)(x, p, ctx->stream); break;
        }
    };
    const char* const too_many = "kv_attention: too many tokens a sequence for one call";
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
    if (blocks == nullptr && rows > kFewRows &&
        all_rows / kWideRows * cache->kv_heads >= static_cast<uint64_t>(ctx->compute_units)) {
        AttendPlan p{};
        p.wide = true;
        const uint64_t row_tiles = (rows + kWideRows - 1) / kWideRows;
        if (row_tiles > 65535) return ctx->fail(GOFANN_ERR_UNSUPPORTED, too_many);
        a.splits = 1;
        a.split_tiles = static_cast<int>(most_tiles);
        a.row_tiles = static_cast<int>(row_tiles);
        const bool mixed = static_cast<uint64_t>(batch->sequences) * tokens > batch->queries;
        a.rows_over = mixed ? kFewRows : 0;
        p.grid = dim3(cache->kv_heads, static_cast<uint32_t>(row_tiles), batch->sequences);
        launch(a, p);
        if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_attention: launch");
        if (!mixed) return GOFANN_OK;
        a.rows_over = 0;
        a.rows_upto = kFewRows;
        rows = kFewRows;
        if (static_cast<uint64_t>(batch->sequences) * kFewRows < part_rows) {
            a.part_rows = kFewRows;
            part_rows = static_cast<uint64_t>(batch->sequences) * kFewRows;
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
    if (row_tiles > 65535) return ctx->fail(GOFANN_ERR_UNSUPPORTED, too_many);
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
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_attention: launch");
    return GOFANN_OK;
}

}  // namespace gofann
