// kv_read.hip -- tokens' keys and values out of the paged 4-bit key/value cache.
#include "kv_common.hpp"

namespace gofann {
namespace kv {
namespace {

struct ReadArgs {
    Batch batch;
    Rows k, v;  // either may be missing
    const uint8_t* k_codes;
    const uint8_t* k_scales;
    const uint8_t* v_codes;
    const uint8_t* v_scales;
};

// The inverse of append, and cut up as it is: a workgroup takes one page of one
// key/value head, D / 8 threads a row, eight channels a thread, so that a row
// is written in whole lines.  Exact: a code times its group's power of two is
// an element.  Tokens without a page get zeros.  HBM bounds it: 30,005 tokens of 8
// heads of 128 channels (127 MB) take 32 us, 3.9 TB/s, and 22.5 alternating between
// two states.
template <class E, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a)
{
    constexpr int kLanes = D / 8;
    constexpr int kTokens = 256 / kLanes;
    const Batch& t = a.batch;
    const int P = 1 << t.page_shift;
    const int h = blockIdx.x, b = blockIdx.z;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    if (n == 0) return;
    // Below 0 where the batch has more tokens than positions: blocks before the
    // first have no page, as blocks past the table have none.
    const int start = len - n;
    const int block = (start >> t.page_shift) + static_cast<int>(blockIdx.y);
    // Compared as blocks: behind a length near 2^31 the position would wrap.
    if (block > (len - 1) >> t.page_shift) return;
    const int page_begin = block * P;
    const int page = t.page(b, block);
    const int from = start > page_begin ? start - page_begin : 0;
    const int there = len - page_begin < P ? len - page_begin : P;
    const int held_to = page < 0 ? 0 : t.max_positions - page_begin;  // positions that are read

    const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
    const int64_t ph = static_cast<int64_t>(page < 0 ? 0 : page) * t.kv_heads + h;
    const uint8_t* const kc = a.k_codes + ph * P * (D / 2);
    const uint8_t* const ks = a.k_scales + ph * P * (D / 32);
    const uint8_t* const vc = a.v_codes + ph * P * (D / 2);
    const uint8_t* const vs = a.v_scales + ph * P * (D / 32);
#pragma unroll 4
    for (int s = from + row; s < there; s += kTokens) {
        const int64_t q = q0 + (page_begin + s - start);
        const bool in = s < held_to;
        if (a.k.p != nullptr) {
            u32x4 x{0, 0, 0, 0};
            if (in)
                x = held<E>(*reinterpret_cast<const uint32_t*>(kc + s * (D / 2) + 4 * lane),
                            ks[s * (D / 32) + lane / 4]);
            store8(a.k.p + q * a.k.token_stride + h * a.k.head_stride + 8 * lane, x, a.k.wide);
        }
        if (a.v.p != nullptr) {
            u32x4 x{0, 0, 0, 0};
            if (in) {
                const uint8_t* const v8 = vc + (s / 8) * (4 * D) + (s % 8) * (D / 32);
                uint32_t codes;
                if constexpr (D == 64)
                    codes = *reinterpret_cast<const uint16_t*>(v8 + (2 * lane) * (D / 4)) |
                            static_cast<uint32_t>(
                                *reinterpret_cast<const uint16_t*>(v8 + (2 * lane + 1) * (D / 4)))
                                << 16;
                else if constexpr (D == 128)
                    codes = *reinterpret_cast<const uint32_t*>(v8 + lane * (D / 4));
                else
                    codes = *reinterpret_cast<const uint32_t*>(v8 + (lane / 2) * (D / 4) + 4 * (lane % 2));
                x = held<E>(codes, vs[((s / 8) * (D / 32) + lane / 4) * 8 + s % 8]);
            }
            store8(a.v.p + q * a.v.token_stride + h * a.v.head_stride + 8 * lane, x, a.v.wide);
        }
    }
}

template <class E>
void launch(const ReadArgs& a, uint32_t dim, dim3 grid, hipStream_t stream)
{
    switch (dim) {
        case 64: kv_read_kernel<E, 64><<<grid, 256, 0, stream>>>(a); break;
        case 128: kv_read_kernel<E, 128><<<grid, 256, 0, stream>>>(a); break;
        default: kv_read_kernel<E, 256><<<grid, 256, 0, stream>>>(a); break;
    }
}

}  // namespace
}  // namespace kv

int kv_read(Context* ctx, const gofann_kv_cache* cache, const gofann_kv_batch* batch,
            const gofann_kv_rows* k, const gofann_kv_rows* v)
{
    using namespace kv;
    const ReadArgs a{batch_of(cache, batch), rows_of(k),      rows_of(v),     cache->k_codes,
                     cache->k_scales,        cache->v_codes,  cache->v_scales};
    const uint64_t tokens = batch->query_offsets == nullptr ? 1 : batch->max_queries;
    const uint64_t touched = (tokens + cache->page_size - 2) / cache->page_size + 1;
    if (touched > 65535)
        return ctx->fail(GOFANN_ERR_UNSUPPORTED, "kv_read: too many tokens a sequence for one call");
    const dim3 grid(cache->kv_heads, static_cast<uint32_t>(touched), batch->sequences);
    if (cache->elem == GOFANN_ELEM_BF16)
        launch<Bf16>(a, cache->dim, grid, ctx->stream);
    else
        launch<F16>(a, cache->dim, grid, ctx->stream);
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_read: launch");
    return GOFANN_OK;
}

}  // namespace gofann
