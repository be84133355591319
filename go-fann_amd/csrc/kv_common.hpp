// kv_common.hpp -- what the kernels of the paged 4-bit key/value cache share:
// argument blocks, element types, the 4-bit conversions and lookups of a
// sequence's length, tokens and pages.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

#include "gofann_internal.hpp"

namespace gofann {
namespace kv {

using f32x4 = float __attribute__((ext_vector_type(4)));
using f32x16 = float __attribute__((ext_vector_type(16)));
using i32x4 = int __attribute__((ext_vector_type(4)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using u32x2 = uint32_t __attribute__((ext_vector_type(2)));

// Positions a wave takes at once: a tile never crosses a page (pages hold a
// power of two of at least 32 positions) and one word of the filter covers it.
constexpr int kTile = 32;

// The 16-bit element types of queries, keys, values and outputs.
struct Bf16 {
    using T = __bf16;
    using V2 = __bf16 __attribute__((ext_vector_type(2)));
    using V8 = __bf16 __attribute__((ext_vector_type(8)));
    static constexpr int kMinExp = -125, kMaxExp = 125;  // a group's exponents
    static constexpr float kRaise = 0.0f;  // of attention weights, in powers of two
    static __device__ f32x4 mfma(V8 a, V8 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ f32x16 mfma(V8 a, V8 b, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    // Byte SEL of `codes` as two elements times the power of two in bits 30:23
    // of `scale` (the conversion reads no other bit of it; exact).
    template <int SEL>
    static __device__ uint32_t decode(uint32_t codes, uint32_t scale)
    {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                                codes, __builtin_bit_cast(float, scale), SEL));
    }
};
struct F16 {
    using T = _Float16;
    using V2 = _Float16 __attribute__((ext_vector_type(2)));
    using V8 = _Float16 __attribute__((ext_vector_type(8)));
    // Every code times 2^e in this range is a finite f16, without rounding.
    static constexpr int kMinExp = -23, kMaxExp = 13;
    static constexpr float kRaise = 7.0f;
    static __device__ f32x4 mfma(V8 a, V8 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ f32x16 mfma(V8 a, V8 b, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    template <int SEL>
    static __device__ uint32_t decode(uint32_t codes, uint32_t scale)
    {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(
                                                codes, __builtin_bit_cast(float, scale), SEL));
    }
};

// f(integral_constant<int, 0>), .. f(integral_constant<int, N - 1>).
template <int... I, class F>
__device__ __forceinline__ void each_impl(std::integer_sequence<int, I...>, F&& f)
{
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f)
{
    each_impl(std::make_integer_sequence<int, N>{}, static_cast<F&&>(f));
}

// Rows of 16-bit elements: row (token, head) at p + token * token_stride +
// head * head_stride (in elements); `wide`: every row starts at a multiple of
// 16 bytes.
struct Rows {
    uint16_t* p;
    int64_t token_stride;
    int64_t head_stride;
    int wide;
};

inline Rows rows_of(const gofann_kv_rows* r)
{
    if (r == nullptr || r->data == nullptr) return Rows{nullptr, 0, 0, 0};
    const bool wide = (reinterpret_cast<uintptr_t>(r->data) % 16 == 0) && r->token_stride % 8 == 0 &&
                      r->head_stride % 8 == 0;
    return Rows{static_cast<uint16_t*>(r->data), r->token_stride, r->head_stride, wide ? 1 : 0};
}

__device__ __forceinline__ u32x4 load8(const uint16_t* p, int wide)
{
    if (wide) return *reinterpret_cast<const u32x4*>(p);
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = static_cast<uint32_t>(p[2 * i]) | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
    return v;
}

__device__ __forceinline__ void store8(uint16_t* p, u32x4 v, int wide)
{
    if (wide) {
        *reinterpret_cast<u32x4*>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p[2 * i] = static_cast<uint16_t>(v[i]);
        p[2 * i + 1] = static_cast<uint16_t>(v[i] >> 16);
    }
}

// The batch as the kernels read it.  Every value that comes from device
// memory (lengths, offsets, page ids) is clamped or checked before it is
// used in an address.
struct Batch {
    const int32_t* page_table;
    const int32_t* lengths;
    const int32_t* query_offsets;
    const uint32_t* visible;
    int64_t table_stride;
    int64_t visible_stride;
    int64_t visible_width;   // words of a row that are read
    int table_width;
    int queries;
    int page_shift;  // log2 of the page size
    int pages;
    int kv_heads;
    int max_positions;  // positions from here on have no page

    // Positions of sequence b, those without a page among them: its tokens are
    // the last ones, wherever its page table ends.
    __device__ int length(int b) const
    {
        const int n = lengths[b];
        return n < 0 ? 0 : n;
    }
    // First row of sequence b's tokens and their number.
    __device__ int first_query(int b) const
    {
        if (query_offsets == nullptr) return b;
        const int n = query_offsets[b];
        return n < 0 ? 0 : n > queries ? queries : n;
    }
    __device__ int new_tokens(int b, int first) const
    {
        if (query_offsets == nullptr) return first < queries ? 1 : 0;
        int n = query_offsets[b + 1];
        n = n > queries ? queries : n;
        return n > first ? n - first : 0;
    }
    // Page of block j of sequence b, -1 where there is none.
    __device__ int page(int b, int j) const
    {
        if (j < 0 || j >= table_width) return -1;
        const int p = page_table[b * table_stride + j];
        return p >= 0 && p < pages ? p : -1;
    }
    // The filter's word of positions [32 w, 32 w + 32).
    __device__ uint32_t word(int b, int w) const
    {
        if (visible == nullptr) return 0xFFFFFFFFu;
        return w < visible_width ? visible[b * visible_stride + w] : 0u;
    }
};

inline Batch batch_of(const gofann_kv_cache* c, const gofann_kv_batch* b)
{
    int shift = 0;
    while ((1u << shift) < c->page_size) ++shift;
    const uint64_t fits = static_cast<uint64_t>(b->table_width) << shift;
    const uint64_t most = b->max_length < fits ? b->max_length : fits;
    return Batch{b->page_table,
                 b->lengths,
                 b->query_offsets,
                 b->visible,
                 static_cast<int64_t>(b->table_stride),
                 static_cast<int64_t>(b->visible_stride),
                 static_cast<int64_t>(b->visible_width != 0 ? b->visible_width : b->visible_stride),
                 static_cast<int>(b->table_width),
                 static_cast<int>(b->queries),
                 shift,
                 static_cast<int>(c->pages),
                 static_cast<int>(c->kv_heads),
                 static_cast<int>(most)};
}

}  // namespace kv
}  // namespace gofann
