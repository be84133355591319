// kv_settle.hip -- drafts of tokens over the paged 4-bit key/value cache, apart
// from their attention: the bits and depths of a draft's tree, the path through
// it that a model's answers accept, and that path's keys and values moved to
// the positions right behind the sequence's earlier ones.
#include "kv_common.hpp"

namespace gofann {
namespace kv {
namespace {

// Tokens of a tree whose parents a workgroup holds in LDS (32 KB).
constexpr int kTreeTokens = 8192;

struct TreeArgs {
    Batch batch;
    const int32_t* parents;
    uint32_t* sees;   // [queries][words] or NULL
    int32_t* depths;  // [queries] or NULL
    int words;
};

// A thread a token: the walk from it to its root goes to ever lower tokens, so
// its words are finished from the highest down and each is written once.  The
// parents up to the workgroup's last token are in LDS; a step of the walk is
// one read of it.  40 tokens for each of 64 sequences take 3.4 us, mostly the
// launch and the chain of offsets and parents.
__global__ __launch_bounds__(256) void kv_tree_kernel(TreeArgs a)
{
    __shared__ int32_t parent[kTreeTokens];
    const Batch& t = a.batch;
    const int b = blockIdx.y;
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    const int begin = blockIdx.x * 256;
    if (begin >= n) return;
    const int stop = n < begin + 256 ? n : begin + 256;
    for (int i = threadIdx.x; i < stop; i += 256) {
        const int p = a.parents[q0 + i];
        parent[i] = p >= 0 && p < i ? p : -1;
    }
    __syncthreads();
    const int i = begin + threadIdx.x;
    if (i >= stop) return;
    uint32_t* const row = a.sees + static_cast<int64_t>(q0 + i) * a.words;
    int w = i >> 5, depth = 0;
    uint32_t bits = 1u << (i & 31);
    if (a.sees != nullptr)
        for (int z = w + 1; z < a.words; ++z) row[z] = 0;
    const auto put = [&](int to) {  // word w, and zeros down to word `to`
        if (a.sees == nullptr) return;
        if (w < a.words) row[w] = bits;
        for (int z = w - 1; z > to; --z)
            if (z < a.words) row[z] = 0;
    };
    for (int p = parent[i]; p >= 0; p = parent[p]) {
        ++depth;
        if (p >> 5 != w) {
            put(p >> 5);
            w = p >> 5;
            bits = 0;
        }
        bits |= 1u << (p & 31);
    }
    put(-1);
    if (a.depths != nullptr) a.depths[q0 + i] = depth;
}

struct AcceptArgs {
    Batch batch;
    const int32_t* parents;
    const int32_t* drafted;
    const int32_t* chosen;
    int32_t* path;     // [sequences][width]
    int32_t* lengths;  // [sequences] or NULL
    int32_t* next;     // [sequences] or NULL
    int width;
};

// A wave a sequence.  A child's index is above its parent's, so one pass over
// the tokens, 64 at a time, finds the whole path: of those past the path's last
// token, the lowest that is its child and drafted its answer, again and again
// until the 64 hold none.  A step is a comparison a lane and a ballot; 64
// sequences of up to 40 tokens take 3.2 us.
__global__ __launch_bounds__(64) void kv_accept_kernel(AcceptArgs a)
{
    const Batch& t = a.batch;
    const int lane = threadIdx.x;
    const int b = blockIdx.x;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    int32_t* const path = a.path + static_cast<int64_t>(b) * a.width;
    int count = 0, cur = -1, answer = -1;
    for (int base = 0; base < n && count < a.width; base += 64) {
        const int i = base + lane;
        const bool in = i < n;
        const int parent = in ? a.parents[q0 + i] : -1;
        const int drafted = in ? a.drafted[q0 + i] : 0;
        const int chosen = in ? a.chosen[q0 + i] : 0;
        uint64_t hit = base == 0 ? 1 : 0;  // token 0 is the model's own
        while (count < a.width) {
            if (hit == 0) {
                if (cur < 0) break;
                hit = __ballot(in && i > cur && parent == cur && drafted == answer);
                if (hit == 0) break;
            }
            const int at = __builtin_ctzll(hit);
            hit = 0;
            cur = base + at;
            answer = __builtin_amdgcn_readlane(chosen, at);
            if (lane == 0) path[count] = cur;
            ++count;
        }
    }
    for (int i = count + lane; i < a.width; i += 64) path[i] = -1;
    if (lane != 0) return;
    const int64_t kept = static_cast<int64_t>(len) - n + count;
    if (a.lengths != nullptr) a.lengths[b] = kept < 0 ? 0 : static_cast<int32_t>(kept);
    if (a.next != nullptr) a.next[b] = answer;
}

struct KeepArgs {
    Batch batch;
    const int32_t* path;
    int width;
    uint8_t* k_codes;
    uint8_t* k_scales;
    uint8_t* v_codes;
    uint8_t* v_scales;
    int8_t* box;
    uint8_t* box_scale;
};

// A workgroup moves one sequence's rows of one key/value head and renews its
// boxes, so that reads and writes of a row never meet in two workgroups.  The
// path ascends: the i-th row comes from a token of at least i, so rows of later
// turns lie past everything that an earlier turn wrote, and a turn's rows are
// all in registers before any is written.  D / 8 threads a row, as append has.
//
// Latency bounds it: 64 sequences of 8 heads of 128 channels, up to 10 rows moved
// and a page's keys read for its box, take 6.9 us: offsets and path, page ids,
// rows, then keys, one after another.
template <class E, int D>
__global__ __launch_bounds__(256) void kv_keep_kernel(KeepArgs a)
{
    constexpr int kLanes = D / 8;
    constexpr int kTokens = 256 / kLanes;
    __shared__ float most[kTokens][D], least[kTokens][D];
    __shared__ float amax_part[4];
    __shared__ int first_bad;
    const Batch& t = a.batch;
    const int h = blockIdx.x, b = blockIdx.y;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    if (n == 0) return;
    const int start = len - n;  // below 0 where the batch has more tokens than positions
    const int32_t* const path = a.path + static_cast<int64_t>(b) * a.width;

    // The path ends where it no longer ascends within the draft.
    const int most_kept = a.width < n ? a.width : n;
    if (threadIdx.x == 0) first_bad = most_kept;
    __syncthreads();
    int count = most_kept;
    for (int base = 0; base < most_kept; base += 256) {
        const int i = base + threadIdx.x;
        if (i < most_kept) {
            const int at = path[i], before = i > 0 ? path[i - 1] : -1;
            if (at <= before || at < 0 || at >= n) atomicMin(&first_bad, i);
        }
        __syncthreads();
        count = first_bad;
        __syncthreads();
        if (count < base + 256) break;
    }

    const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
    const int P = 1 << t.page_shift;
    const auto head_of = [&](int page) { return static_cast<int64_t>(page) * t.kv_heads + h; };
    for (int base = 0; base < count; base += kTokens) {
        const int i = base + row;
        int from = -1, to = -1;
        int64_t from_head = -1, to_head = -1;
        if (i < count && path[i] != i) {
            const int src = start + path[i], dst = start + i;
            if (dst >= 0 && src < t.max_positions) {
                const int sp = t.page(b, src >> t.page_shift), dp = t.page(b, dst >> t.page_shift);
                if (sp >= 0 && dp >= 0) {
                    from_head = head_of(sp);
                    to_head = head_of(dp);
                    from = src & (P - 1);
                    to = dst & (P - 1);
                }
            }
        }
        uint32_t kc = 0, vc = 0;
        uint8_t ks = 0, vs = 0;
        // Where a row's values lie: those of eight tokens by unit, D / 32 bytes each.
        const auto value_at = [&](int64_t head, int s) {
            return head * P * (D / 2) + (s / 8) * (4 * D) + (s % 8) * (D / 32);
        };
        const auto value_scale_at = [&](int64_t head, int s) {
            return head * P * (D / 32) + ((s / 8) * (D / 32) + lane / 4) * 8 + s % 8;
        };
        if (from >= 0) {
            kc = *reinterpret_cast<const uint32_t*>(a.k_codes + (from_head * P + from) * (D / 2) + 4 * lane);
            ks = a.k_scales[(from_head * P + from) * (D / 32) + lane / 4];
            const uint8_t* const v = a.v_codes + value_at(from_head, from);
            if constexpr (D == 64)
                vc = *reinterpret_cast<const uint16_t*>(v + (2 * lane) * (D / 4)) |
                     static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(v + (2 * lane + 1) * (D / 4))) << 16;
            else if constexpr (D == 128)
                vc = *reinterpret_cast<const uint32_t*>(v + lane * (D / 4));
            else
                vc = *reinterpret_cast<const uint32_t*>(v + (lane / 2) * (D / 4) + 4 * (lane % 2));
            vs = a.v_scales[value_scale_at(from_head, from)];
        }
        __syncthreads();
        if (from >= 0) {
            *reinterpret_cast<uint32_t*>(a.k_codes + (to_head * P + to) * (D / 2) + 4 * lane) = kc;
            uint8_t* const v = a.v_codes + value_at(to_head, to);
            if constexpr (D == 64) {
                *reinterpret_cast<uint16_t*>(v + (2 * lane) * (D / 4)) = static_cast<uint16_t>(vc);
                *reinterpret_cast<uint16_t*>(v + (2 * lane + 1) * (D / 4)) = static_cast<uint16_t>(vc >> 16);
            } else if constexpr (D == 128) {
                *reinterpret_cast<uint32_t*>(v + lane * (D / 4)) = vc;
            } else {
                *reinterpret_cast<uint32_t*>(v + (lane / 2) * (D / 4) + 4 * (lane % 2)) = vc;
            }
            if (lane % 4 == 0) {
                a.k_scales[(to_head * P + to) * (D / 32) + lane / 4] = ks;
                a.v_scales[value_scale_at(to_head, to)] = vs;
            }
        }
    }
    if (a.box == nullptr) return;

    // Boxes of the pages from the draft's first position to the last one kept.
    int stop = start + count;
    if (stop > t.max_positions) stop = t.max_positions;
    for (int page_begin = (start < 0 ? 0 : start) & ~(P - 1); page_begin < stop; page_begin += P) {
        __syncthreads();  // rows are written, LDS is free again
        const int page = t.page(b, page_begin >> t.page_shift);
        if (page < 0) continue;
        const int there = stop - page_begin < P ? stop - page_begin : P;
        const uint8_t* const kc = a.k_codes + head_of(page) * P * (D / 2);
        const uint8_t* const ks = a.k_scales + head_of(page) * P * (D / 32);
        float hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hi[i] = -__builtin_inff();
            lo[i] = __builtin_inff();
        }
#pragma unroll 4
        for (int s = row; s < there; s += kTokens) {
            const u32x4 x = held<E>(*reinterpret_cast<const uint32_t*>(kc + s * (D / 2) + 4 * lane),
                                    ks[s * (D / 32) + lane / 4]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = static_cast<float>(
                    __builtin_bit_cast(typename E::V2, static_cast<uint32_t>(x[i / 2]))[i % 2]);
                hi[i] = fmaxf(hi[i], f);
                lo[i] = fminf(lo[i], f);
            }
        }
        join_box<D>(hi, lo, most, least, amax_part, a.box + head_of(page) * 2 * D,
                    a.box_scale + head_of(page));
    }
}

template <class E>
void launch_keep(const KeepArgs& a, uint32_t dim, dim3 grid, hipStream_t stream)
{
    switch (dim) {
        case 64: kv_keep_kernel<E, 64><<<grid, 256, 0, stream>>>(a); break;
        case 128: kv_keep_kernel<E, 128><<<grid, 256, 0, stream>>>(a); break;
        default: kv_keep_kernel<E, 256><<<grid, 256, 0, stream>>>(a); break;
    }
}

uint32_t tokens_of(const gofann_kv_batch* batch)
{
    return batch->query_offsets == nullptr ? 1 : batch->max_queries;
}

}  // namespace
}  // namespace kv

int kv_draft_tree(Context* ctx, const gofann_kv_batch* batch, const int32_t* parents, uint32_t words,
                  uint32_t* out_sees, int32_t* out_depths)
{
    using namespace kv;
    if (tokens_of(batch) > static_cast<uint32_t>(kTreeTokens))
        return ctx->fail(GOFANN_ERR_UNSUPPORTED, "kv_draft_tree: at most 8192 tokens a tree");
    const TreeArgs a{rows_only(batch), parents, out_sees, out_depths, static_cast<int>(words)};
    kv_tree_kernel<<<dim3((tokens_of(batch) + 255) / 256, batch->sequences), 256, 0, ctx->stream>>>(a);
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_draft_tree: launch");
    return GOFANN_OK;
}

int kv_draft_accept(Context* ctx, const gofann_kv_batch* batch, const int32_t* parents,
                    const int32_t* drafted, const int32_t* chosen, uint32_t width, int32_t* out_path,
                    int32_t* out_lengths, int32_t* out_next)
{
    using namespace kv;
    AcceptArgs a{rows_only(batch), parents, drafted, chosen, out_path, out_lengths, out_next,
                 static_cast<int>(width)};
    if (tokens_of(batch) == 0) a.batch.queries = 0;  // the arrays may be missing, whatever the offsets say
    kv_accept_kernel<<<batch->sequences, 64, 0, ctx->stream>>>(a);
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_draft_accept: launch");
    return GOFANN_OK;
}

int kv_keep(Context* ctx, const gofann_kv_cache* cache, const gofann_kv_batch* batch,
            const int32_t* path, uint32_t width)
{
    using namespace kv;
    const KeepArgs a{batch_of(cache, batch), path,            static_cast<int>(width),
                     cache->k_codes,         cache->k_scales, cache->v_codes,
                     cache->v_scales,        cache->box,      cache->box_scale};
    const dim3 grid(cache->kv_heads, batch->sequences);
    if (cache->elem == GOFANN_ELEM_BF16)
        launch_keep<Bf16>(a, cache->dim, grid, ctx->stream);
    else
        launch_keep<F16>(a, cache->dim, grid, ctx->stream);
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_keep: launch");
    return GOFANN_OK;
}

}  // namespace gofann
