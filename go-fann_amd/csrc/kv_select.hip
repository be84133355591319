// kv_select.hip -- the blocks of the paged 4-bit key/value cache that each
// token and key/value head reads: integer scores of the queries against the
// pages' boxes, then the highest `width` of them in ascending order.
#include "kv_common.hpp"

namespace gofann {
namespace kv {
namespace {

constexpr int kChunkTiles = 16;               // 16-block tiles a workgroup scores
constexpr int kChunk = 16 * kChunkTiles;      // blocks of them
constexpr uint32_t kForced = 0xFFFFFFFFu;     // above every score's key
constexpr uint32_t kIneligible = 0;           // below every score's key

struct SelectArgs {
    Batch batch;
    Rows q;
    const int8_t* box;
    const uint8_t* box_scale;
    uint32_t* keys;  // [queries][kv_heads][key_stride]
    int64_t key_stride;
    int32_t* out;
    int group;        // heads a key/value head
    int group_shift;  // log2 of the rows a token's heads take of a 16-row tile
    int head_tiles;   // 16-row tiles of one token's heads, where they are more than 16
    int width, first, last;
};

// Position of token i of sequence b, and the blocks up to it; none below 0.
__device__ __forceinline__ int position(int len, int n, int i) { return len - n + i; }

// Whether block j (page_size positions) has a visible position up to pos.
__device__ __forceinline__ bool any_visible(const Batch& t, int b, int j, int pos)
{
    if (t.visible == nullptr) return true;
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

// Scores.  The rows of an i8 product are a token's heads (each token padded
// to a power of two of rows by repeating its last head, which changes no
// maximum), the columns blocks: a lane then holds four heads of one block,
// and the maximum over a token's heads stays in the lane and its neighbours
// 16 and 32 lanes away.  sum_c max(q most, q least) is one product of length
// 2 dim, of the positive part of q with `most` and the negative with `least`.
template <class E, int D>
__global__ __launch_bounds__(256) void kv_score_kernel(SelectArgs a)
{
    constexpr int K = D / 64;  // products of 64 channels
    const Batch& t = a.batch;
    const int h = blockIdx.x % t.kv_heads;
    const int chunk = blockIdx.x / t.kv_heads;
    const int b = blockIdx.z;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    const int rows_shift = a.group_shift;             // rows a token takes: 1 << rows_shift
    const int tokens = 16 >> rows_shift;
    const int i0 = blockIdx.y * tokens;
    if (i0 >= n) return;
    const int i_last = (i0 + tokens < n ? i0 + tokens : n) - 1;
    const int last_pos = position(len, n, i_last);
    if (last_pos < 0) return;
    const int blocks = (last_pos >> t.page_shift) + 1;
    if (chunk * kChunk >= blocks) return;

    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int r16 = lane % 16, g4 = lane / 16;

    // Positive and negative part of the quantized queries, 16 channels a lane
    // and product; the rows' powers of two.
    const auto load_queries = [&](int ht, i32x4 (&pos)[K], i32x4 (&neg)[K], float (&unit)[4]) {
        const int i = i0 + (r16 >> rows_shift);
        int head = 16 * ht + (r16 & ((1 << rows_shift) - 1));
        head = head < a.group ? head : a.group - 1;
        const int token = i < n ? i : n - 1;
        const uint16_t* const row = a.q.p + (q0 + token) * a.q.token_stride +
                                    (static_cast<int64_t>(h) * a.group + head) * a.q.head_stride;
        float x[K][16];
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const u32x4 v = load8(row + 64 * k + 16 * g4 + 8 * half, a.q.wide);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float f = static_cast<float>(
                        __builtin_bit_cast(typename E::V2, static_cast<uint32_t>(v[j / 2]))[j % 2]);
                    f = f != f ? 0.0f : f;
                    const float m = __builtin_fabsf(f);
                    amax = m > amax && m < __builtin_inff() ? m : amax;
                    x[k][8 * half + j] = f;
                }
            }
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        int e = amax > 0.0f ? __builtin_amdgcn_frexp_expf(amax) - 7 : -125;
        e = e < -125 ? -125 : e > 125 ? 125 : e;
        const float inv = __builtin_bit_cast(float, static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t p = 0, m = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float f = __builtin_rintf(x[k][4 * w + j] * inv);
                    f = f > 127.0f ? 127.0f : f < -127.0f ? -127.0f : f;
                    const int v = static_cast<int>(f);
                    p |= static_cast<uint32_t>(v > 0 ? v : 0) << (8 * j);
                    m |= static_cast<uint32_t>((v < 0 ? v : 0) & 255) << (8 * j);
                }
                pos[k][w] = static_cast<int>(p);
                neg[k][w] = static_cast<int>(m);
            }
        const float mine = __builtin_bit_cast(float, static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) unit[i4] = __shfl(mine, 4 * g4 + i4);
    };

    i32x4 qp[K], qn[K];
    float unit[4];
    load_queries(0, qp, qn, unit);

    for (int tile = wave; tile < kChunkTiles; tile += 4) {
        const int block = chunk * kChunk + 16 * tile + r16;
        if (chunk * kChunk + 16 * tile >= blocks) break;
        const int page = block < blocks ? t.page(b, block) : -1;
        i32x4 hi[K] = {}, lo[K] = {};
        float eb = 0.0f;
        if (page >= 0) {
            const int64_t ph = static_cast<int64_t>(page) * t.kv_heads + h;
            const int8_t* const p = a.box + ph * 2 * D + 16 * g4;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                hi[k] = *reinterpret_cast<const i32x4*>(p + 64 * k);
                lo[k] = *reinterpret_cast<const i32x4*>(p + D + 64 * k);
            }
            eb = __builtin_bit_cast(float, static_cast<uint32_t>(a.box_scale[ph]) << 23);
        }
        float s[4];
        for (int ht = 0; ht < a.head_tiles; ++ht) {
            if (a.head_tiles > 1) load_queries(ht, qp, qn, unit);
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < K; ++k) {
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qp[k], hi[k], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qn[k], lo[k], acc, 0, 0, 0);
            }
            // |acc| < 2^23, so the conversion and both products are exact
            // wherever the result is a normal number.
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = static_cast<float>(acc[i]) * unit[i] * eb;
                s[i] = ht == 0 ? f : fmaxf(s[i], f);
            }
        }
        // Maximum over a token's rows.
        if (rows_shift >= 1) {
            s[0] = s[1] = fmaxf(s[0], s[1]);
            s[2] = s[3] = fmaxf(s[2], s[3]);
        }
        if (rows_shift >= 2) s[0] = s[1] = s[2] = s[3] = fmaxf(s[0], s[2]);
        if (rows_shift >= 3) s[0] = fmaxf(s[0], __shfl_xor(s[0], 16));
        if (rows_shift >= 4) s[0] = fmaxf(s[0], __shfl_xor(s[0], 32));
        const int step = rows_shift >= 2 ? 4 : 1 << rows_shift;  // rows of this lane a token
        if (rows_shift >= 3 && (4 * g4 & ((1 << rows_shift) - 1)) != 0) continue;
        for (int i = 0; i < 4; i += step) {
            const int token = i0 + ((4 * g4 + i) >> rows_shift);
            if (token >= n) break;
            const int pos = position(len, n, token);
            const int mine = pos < 0 ? 0 : (pos >> t.page_shift) + 1;
            if (block >= mine) continue;
            uint32_t key = kIneligible;
            if (page >= 0 && any_visible(t, b, block, pos)) {
                const uint32_t u = __builtin_bit_cast(uint32_t, s[i] + 0.0f);  // -0 as 0
                key = (u & 0x80000000u) ? ~u : u | 0x80000000u;
                if (block < a.first || block >= mine - a.last) key = kForced;
            }
            a.keys[(static_cast<int64_t>(q0 + token) * t.kv_heads + h) * a.key_stride + block] = key;
        }
    }
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)
{
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// The `width` highest keys of a token and head, written in ascending order of
// their blocks: a radix descent finds the least key taken and how many of the
// blocks that have it are, then every thread places its own run of blocks.
__global__ __launch_bounds__(256) void kv_pick_kernel(SelectArgs a)
{
    __shared__ uint32_t hist[256];
    __shared__ uint32_t found[2];
    __shared__ uint32_t part[2][4];
    const Batch& t = a.batch;
    const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    if (i >= n) return;
    const int pos = position(len, n, i);
    const int blocks = pos < 0 ? 0 : (pos >> t.page_shift) + 1;
    const int64_t row = static_cast<int64_t>(q0 + i) * t.kv_heads + h;
    const uint32_t* const keys = a.keys + row * a.key_stride;
    int32_t* const out = a.out + row * a.width;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;

    uint32_t prefix = 0, mask = 0;
    uint32_t want = a.width;  // still to be taken among keys that match the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < blocks; j += 256) {
            const uint32_t k = keys[j];
            if (k != kIneligible && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // Lane l takes the bins 255 - 4 l .. 252 - 4 l, highest first.
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                c[m] = hist[255 - 4 * lane - m];
                sum += c[m];
            }
            const uint32_t incl = wave_scan(sum);
            uint32_t above = incl - sum;
            if (lane == 63 && incl < want) {  // fewer than wanted: all of them
                found[0] = 256;
                found[1] = 0;
            }
            if (above < want && incl >= want) {
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    if (above < want && above + c[m] >= want) {
                        found[0] = 255 - 4 * lane - m;
                        found[1] = want - above;
                    }
                    above += c[m];
                }
            }
        }
        __syncthreads();
        if (found[0] == 256) {  // every eligible block (only at the first digit)
            prefix = 1;
            want = 0;
            mask = 0;
            break;
        }
        prefix |= found[0] << shift;
        mask |= 255u << shift;
        want = found[1];
    }
    // Taken: keys above `prefix`, and the first `want` that equal it.  Where
    // all are taken: keys of at least 1.
    const bool all = mask == 0;
    const int each_thread = (blocks + 255) / 256;
    const int begin = tid * each_thread;
    const int end = begin + each_thread < blocks ? begin + each_thread : blocks;
    uint32_t above = 0, equal = 0;
    for (int j = begin; j < end; ++j) {
        const uint32_t k = keys[j];
        above += all ? k >= prefix : k > prefix;
        equal += !all && k == prefix;
    }
    const uint32_t sa = wave_scan(above), se = wave_scan(equal);
    if (lane == 63) {
        part[0][wave] = sa;
        part[1][wave] = se;
    }
    __syncthreads();
    uint32_t before_a = sa - above, before_e = se - equal, total_a = 0, total_e = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) {
            before_a += part[0][w];
            before_e += part[1][w];
        }
        total_a += part[0][w];
        total_e += part[1][w];
    }
    uint32_t at = before_a + (before_e < want ? before_e : want);
    for (int j = begin; j < end; ++j) {
        const uint32_t k = keys[j];
        bool take = all ? k >= prefix : k > prefix;
        if (!all && k == prefix) {
            take = before_e < want;
            ++before_e;
        }
        if (take) out[at++] = j;
    }
    const uint32_t total = total_a + (total_e < want ? total_e : want);
    for (uint32_t j = total + tid; j < static_cast<uint32_t>(a.width); j += 256) out[j] = -1;
}

template <class E>
void launch_score(const SelectArgs& a, uint32_t dim, dim3 grid, hipStream_t stream)
{
    switch (dim) {
        case 64: kv_score_kernel<E, 64><<<grid, 256, 0, stream>>>(a); break;
        case 128: kv_score_kernel<E, 128><<<grid, 256, 0, stream>>>(a); break;
        default: kv_score_kernel<E, 256><<<grid, 256, 0, stream>>>(a); break;
    }
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
    a.width = static_cast<int>(width);
    a.first = static_cast<int>(first);
    a.last = static_cast<int>(last);
    const uint32_t tokens = batch->query_offsets == nullptr ? 1 : batch->max_queries;
    if (tokens > 65535)
        return ctx->fail(GOFANN_ERR_UNSUPPORTED, "kv_select: at most 65535 tokens a sequence");
    const uint32_t most = static_cast<uint32_t>(a.batch.max_positions);
    const uint32_t blocks = (most + cache->page_size - 1) / cache->page_size;
    a.key_stride = blocks;
    const size_t bytes = static_cast<size_t>(batch->queries) * cache->kv_heads * blocks * 4;
    if (bytes > 0) {
        a.keys = static_cast<uint32_t*>(ctx->workspace(Context::kScratchKv, bytes));
        if (a.keys == nullptr) return GOFANN_ERR_NOMEM;
    }
    if (blocks > 0) {
        const uint32_t per = 16u >> a.group_shift;
        const dim3 grid((blocks + kChunk - 1) / kChunk * cache->kv_heads, (tokens + per - 1) / per,
                        batch->sequences);
        if (cache->elem == GOFANN_ELEM_BF16)
            launch_score<Bf16>(a, cache->dim, grid, ctx->stream);
        else
            launch_score<F16>(a, cache->dim, grid, ctx->stream);
    }
    kv_pick_kernel<<<dim3(cache->kv_heads, tokens, batch->sequences), 256, 0, ctx->stream>>>(a);
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_select: launch");
    return GOFANN_OK;
}

}  // namespace gofann
