// kv_append.hip -- new tokens into the paged 4-bit key/value cache: keys and
// values quantized in groups of 32 channels, and the box of every page that a
// token falls in.
#include "kv_common.hpp"

namespace gofann {
namespace kv {
namespace {

struct AppendArgs {
    Batch batch;
    Rows k, v, k_held, v_held;
    uint8_t* k_codes;
    uint8_t* k_scales;
    uint8_t* v_codes;
    uint8_t* v_scales;
    int8_t* box;
    uint8_t* box_scale;
};

// Eight channels of a row in 32 bits, and the same eight as codes (one dword)
// under their group's exponent.
template <class E>
struct Octet {
    uint32_t codes;
    uint32_t exponent;  // e + 127
};

// A group is four neighbouring lanes' octets.
template <class E>
__device__ __forceinline__ Octet<E> quantize(u32x4 raw)
{
    float x[8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto p = __builtin_bit_cast(typename E::V2, static_cast<uint32_t>(raw[i]));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float f = static_cast<float>(p[j]);
            f = f != f ? 0.0f : f;
            x[2 * i + j] = f;
            const float a = __builtin_fabsf(f);
            amax = a > amax && a < __builtin_inff() ? a : amax;
        }
    }
    amax = fmaxf(amax, __shfl_xor(amax, 1));
    amax = fmaxf(amax, __shfl_xor(amax, 2));
    // amax = m 2^t, 0.5 <= m < 1: the least e with m 2^t <= 0.75 2^(e + 3).
    const int t = __builtin_amdgcn_frexp_expf(amax);
    const float m = __builtin_amdgcn_frexp_mantf(amax);
    int e = m > 0.75f ? t - 2 : t - 3;
    e = e < E::kMinExp ? E::kMinExp : e > E::kMaxExp ? E::kMaxExp : e;
    if (!(amax > 0.0f)) e = E::kMinExp;
    Octet<E> o;
    o.exponent = static_cast<uint32_t>(e + 127);
    const float scale = __builtin_bit_cast(float, o.exponent << 23);
    // The conversion divides by the scale, rounds halfway cases to the even
    // code and saturates, infinities included.
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
    o.codes = c;
    return o;
}

template <class E>
__device__ __forceinline__ u32x4 held(uint32_t codes, uint32_t exponent)
{
    const uint32_t s = exponent << 23;
    return u32x4{E::template decode<0>(codes, s), E::template decode<1>(codes, s),
                 E::template decode<2>(codes, s), E::template decode<3>(codes, s)};
}

// A workgroup takes one page of one key/value head.  Eight channels a thread,
// D / 8 threads a token, 256 / (D / 8) tokens at a time.  With a box to renew
// the page's earlier tokens are decoded again: the box depends on the page's
// codes alone, however they got there.
//
// Traffic bounds it: 15,000 tokens of 8 heads of 128 channels, held values
// returned (148 MB), take 30 us, 4.9 TB/s, what a large copy reaches.  One token
// for each of 64 sequences takes 6.4 us, the latency of looking up the page,
// reading its other keys and joining the box.
template <class E, int D>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a)
{
    constexpr int kLanes = D / 8;
    constexpr int kTokens = 256 / kLanes;
    __shared__ float most[kTokens][D], least[kTokens][D];
    __shared__ float amax_part[4];

    const Batch& t = a.batch;
    const int P = 1 << t.page_shift;
    const int h = blockIdx.x, b = blockIdx.z;
    const int len = t.length(b);
    const int q0 = t.first_query(b);
    const int n = t.new_tokens(b, q0);
    const int start = len - n;  // below 0 where the batch has more tokens than positions
    const int begin = start < 0 ? 0 : start;
    const int block = (begin >> t.page_shift) + static_cast<int>(blockIdx.y);
    if (n == 0 || block >= t.table_width) return;
    const int page_begin = block << t.page_shift;
    const int stop = len < t.max_positions ? len : t.max_positions;
    if (page_begin >= stop || begin >= stop) return;
    const int page = t.page(b, block);
    if (page < 0) return;
    const int fresh = (begin > page_begin ? begin : page_begin) - page_begin;
    const int there = (stop - page_begin < P ? stop - page_begin : P);

    const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
    const int64_t ph = static_cast<int64_t>(page) * t.kv_heads + h;
    uint8_t* const kc = a.k_codes + ph * P * (D / 2);
    uint8_t* const ks = a.k_scales + ph * P * (D / 32);
    uint8_t* const vc = a.v_codes + ph * P * (D / 2);
    uint8_t* const vs = a.v_scales + ph * P * (D / 32);

    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi[i] = -__builtin_inff();
        lo[i] = __builtin_inff();
    }
    const bool boxed = a.box != nullptr;
    for (int base = boxed ? 0 : fresh / kTokens * kTokens; base < there; base += kTokens) {
        const int s = base + row;
        const bool is_new = s >= fresh && s < there;
        const bool is_old = s < fresh;
        Octet<E> ko{0, 0};
        // Whole groups of four lanes are in or out together.
        if (is_new) {
            const int64_t q = q0 + (page_begin + s - start);
            const u32x4 kr = load8(a.k.p + q * a.k.token_stride + h * a.k.head_stride + 8 * lane, a.k.wide);
            const u32x4 vr = load8(a.v.p + q * a.v.token_stride + h * a.v.head_stride + 8 * lane, a.v.wide);
            ko = quantize<E>(kr);
            const Octet<E> vo = quantize<E>(vr);
            *reinterpret_cast<uint32_t*>(kc + s * (D / 2) + 4 * lane) = ko.codes;
            if (lane % 4 == 0) ks[s * (D / 32) + lane / 4] = static_cast<uint8_t>(ko.exponent);
            uint8_t* const v8 = vc + (s / 8) * (16 * D / 4) + (s % 8) * (D / 32);
            if constexpr (D == 64) {
                *reinterpret_cast<uint16_t*>(v8 + (2 * lane) * (D / 4)) = static_cast<uint16_t>(vo.codes);
                *reinterpret_cast<uint16_t*>(v8 + (2 * lane + 1) * (D / 4)) =
                    static_cast<uint16_t>(vo.codes >> 16);
            } else if constexpr (D == 128) {
                *reinterpret_cast<uint32_t*>(v8 + lane * (D / 4)) = vo.codes;
            } else {
                *reinterpret_cast<uint32_t*>(v8 + (lane / 2) * (D / 4) + 4 * (lane % 2)) = vo.codes;
            }
            if (lane % 4 == 0)
                vs[((s / 8) * (D / 32) + lane / 4) * 8 + s % 8] = static_cast<uint8_t>(vo.exponent);
            if (a.k_held.p != nullptr)
                store8(a.k_held.p + q * a.k_held.token_stride + h * a.k_held.head_stride + 8 * lane,
                       held<E>(ko.codes, ko.exponent), a.k_held.wide);
            if (a.v_held.p != nullptr)
                store8(a.v_held.p + q * a.v_held.token_stride + h * a.v_held.head_stride + 8 * lane,
                       held<E>(vo.codes, vo.exponent), a.v_held.wide);
        } else if (is_old && boxed) {
            ko.codes = *reinterpret_cast<const uint32_t*>(kc + s * (D / 2) + 4 * lane);
            ko.exponent = ks[s * (D / 32) + lane / 4];
        }
        if (boxed && s < there) {
            const u32x4 x = held<E>(ko.codes, ko.exponent);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = static_cast<float>(
                    __builtin_bit_cast(typename E::V2, static_cast<uint32_t>(x[i / 2]))[i % 2]);
                hi[i] = fmaxf(hi[i], f);
                lo[i] = fminf(lo[i], f);
            }
        }
    }
    if (!boxed) return;

#pragma unroll
    for (int i = 0; i < 8; ++i) {
        most[row][8 * lane + i] = hi[i];
        least[row][8 * lane + i] = lo[i];
    }
    __syncthreads();
    const int c = threadIdx.x % D;
    float mh = -__builtin_inff(), ml = __builtin_inff();
    for (int r = 0; r < kTokens; ++r) {
        mh = fmaxf(mh, most[r][c]);
        ml = fminf(ml, least[r][c]);
    }
    float amax = fmaxf(__builtin_fabsf(mh), __builtin_fabsf(ml));
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) amax = fmaxf(amax, __shfl_xor(amax, m));
    if (threadIdx.x % 64 == 0) amax_part[threadIdx.x / 64] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(amax_part[0], amax_part[1]), fmaxf(amax_part[2], amax_part[3]));
    // Exact: the values are codes times powers of two, so amax = m 2^t has
    // m 2^7 <= 127, and so is the division by a power of two.
    int e = __builtin_amdgcn_frexp_expf(amax) - 7;
    e = e < -125 ? -125 : e > 125 ? 125 : e;
    if (!(amax > 0.0f)) e = -125;
    const float inv = __builtin_bit_cast(float, static_cast<uint32_t>(127 - e) << 23);
    if (static_cast<int>(threadIdx.x) < D) {
        a.box[ph * 2 * D + c] = static_cast<int8_t>(__builtin_ceilf(mh * inv));
        a.box[ph * 2 * D + D + c] = static_cast<int8_t>(__builtin_floorf(ml * inv));
    }
    if (threadIdx.x == 0) a.box_scale[ph] = static_cast<uint8_t>(e + 127);
}

template <class E>
void launch(const AppendArgs& a, uint32_t dim, dim3 grid, hipStream_t stream)
{
    switch (dim) {
        case 64: kv_append_kernel<E, 64><<<grid, 256, 0, stream>>>(a); break;
        case 128: kv_append_kernel<E, 128><<<grid, 256, 0, stream>>>(a); break;
        default: kv_append_kernel<E, 256><<<grid, 256, 0, stream>>>(a); break;
    }
}

}  // namespace
}  // namespace kv

int kv_append(Context* ctx, const gofann_kv_cache* cache, const gofann_kv_batch* batch,
              const gofann_kv_rows* k, const gofann_kv_rows* v, const gofann_kv_rows* k_held,
              const gofann_kv_rows* v_held)
{
    using namespace kv;
    AppendArgs a{batch_of(cache, batch), rows_of(k),      rows_of(v),      rows_of(k_held),
                 rows_of(v_held),        cache->k_codes,  cache->k_scales, cache->v_codes,
                 cache->v_scales,        cache->box,      cache->box_scale};
    const uint64_t tokens = batch->query_offsets == nullptr ? 1 : batch->max_queries;
    // Pages that so many tokens in a row can touch.
    uint64_t touched = (tokens + cache->page_size - 2) / cache->page_size + 1;
    if (touched > batch->table_width) touched = batch->table_width;
    if (touched == 0) return GOFANN_OK;
    if (touched > 65535)
        return ctx->fail(GOFANN_ERR_UNSUPPORTED, "kv_append: too many tokens a sequence for one call");
    const dim3 grid(cache->kv_heads, static_cast<uint32_t>(touched), batch->sequences);
    if (cache->elem == GOFANN_ELEM_BF16)
        launch<Bf16>(a, cache->dim, grid, ctx->stream);
    else
        launch<F16>(a, cache->dim, grid, ctx->stream);
    if (hipGetLastError() != hipSuccess) return ctx->fail(GOFANN_ERR_HIP, "kv_append: launch");
    return GOFANN_OK;
}

}  // namespace gofann
