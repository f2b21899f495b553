#pragma once
// What the serving entry points share (packed_attention.hip, cache4.hip,
// cache4_attention.hip): rows of 16-bit tensors and the layout of the 4-bit
// key/value cache.

#include "tilemix_device.h"
#include "tilemix_launch.h"

#include <algorithm>
#include <cstdint>

namespace tilemix {

// ------------------------------------------------------------------ tensors

// A [tokens][heads][d] tensor of 16-bit values: elements between tokens and heads.
struct Rows {
    std::int64_t row, head;
};

// Checks and completes the strides (0 = dense) of a tensor whose rows move in
// pieces of `piece` elements. A tensor of no tokens may be null.
inline bool make_rows(Rows& out, const void* data, int tokens, int heads, int d, std::int64_t row_stride,
                      std::int64_t head_stride, int piece) {
    constexpr std::int64_t kMost = std::int64_t{1} << 40;
    out.head = head_stride ? head_stride : d;
    out.row = row_stride ? row_stride : static_cast<std::int64_t>(heads) * d;
    if (tokens > 0 && !data) return false;
    if (reinterpret_cast<std::uintptr_t>(data) % (2 * static_cast<std::size_t>(piece)) != 0) return false;
    if (out.head < 0 || out.row < 0 || out.head > kMost || out.row > kMost || out.head % piece != 0 || out.row % piece != 0)
        return false;
    // No memory holds a tensor that reaches further; strided_heads_ok's products fit 63 bits then.
    constexpr std::int64_t kReach = std::int64_t{1} << 48;
    if (out.row > kReach / std::max(tokens, 1) || out.head > kReach / heads) return false;
    return strided_heads_ok(heads, std::max(tokens, 1), d, out.head, out.row);
}

// Causal rows are aligned at the end of their keys: row i of q_len sees keys 0 .. context + i,
// context = k_len - q_len. The last key that row `row` sees; a row past the end sees what the
// last one does, so that no sum passes 2^31 where k_len is just below it.
__host__ __device__ inline int last_seen(int context, int row, int q_len) {
    return context + (row < q_len ? row : q_len - 1);
}

// -------------------------------------------------------------- 4-bit cache

// A block holds 32 tokens of one key head, in the order in which a wave of the
// attention kernel takes them. With B = ceil(d / 64) groups of 64 features:
//   key codes    [32 tokens][4 g][B m][2 w] words: features 64 m + 16 g + 8 w + e,
//                feature e at bits 4 (e / 2) + 16 (e % 2) of the word
//   value codes  [16 B quarters][32 places] of 16 bits: features 4 quarter + f at bits 4 f
//   key parameters, value parameters   [B][32 places] words: bf16 scale (low half), bf16 minimum
// The value of a code is minimum + scale * code; features past d have code 0.
inline constexpr int kCacheKeys = 32;   // tokens of a block
inline constexpr int kCacheGroup = 64;  // features that share a scale and a minimum
// Scales below this count as 0 (every code 0), so that 1 / scale and the
// remainders of a quotient stay normal numbers.
inline constexpr float kLeastScale = 7.888609052210118e-31f;  // 2^-100

__host__ __device__ constexpr int cache_groups(int d) { return (d + kCacheGroup - 1) / kCacheGroup; }
__host__ __device__ constexpr int cache_block_bytes(int groups) { return kCacheKeys * 72 * groups; }
// Offsets inside a block.
__host__ __device__ constexpr int cache_values_at(int groups) { return 1024 * groups; }
__host__ __device__ constexpr int cache_key_params_at(int groups) { return 2048 * groups; }
__host__ __device__ constexpr int cache_value_params_at(int groups) { return 2176 * groups; }
// Place of token t of a block among the values and parameters: the 8 tokens that
// one lane group of the attention kernel's MFMAs takes lie side by side.
__host__ __device__ constexpr int cache_place(int t) { return 8 * ((t & 15) >> 2) + 4 * (t >> 4) + (t & 3); }

struct Cache {
    std::uint8_t* data;
    std::int64_t pages;
    std::int64_t head_bytes;  // of a page: page_size / 32 blocks
    std::int64_t page_bytes;  // kv_heads * head_bytes
    int page_size;
    int kv_heads;
    int groups;
};

// Where a block lies: bytes from the cache's start (with head 0's part of the page; a head more is
// head_bytes more). `block` is its number in the page. A head's part of a page may pass 2 GiB
// (make_cache: head_bytes under 2^32), so that neither product fits 32 bits.
__host__ __device__ inline std::int64_t cache_block_at(std::int64_t page, std::int64_t page_bytes, int block, int block_bytes) {
    return page * page_bytes + static_cast<std::int64_t>(block) * block_bytes;
}

// TILEMIX_SUCCESS, or the error of the cache arguments.
inline hipError_t make_cache(Cache& out, const std::uint8_t* data, std::int64_t pages, int page_size, int kv_heads, int d) {
    if (!data || reinterpret_cast<std::uintptr_t>(data) % 16 != 0 || pages <= 0 || pages > 0x7fffffffLL || page_size <= 0 ||
        page_size % kCacheKeys != 0 || kv_heads <= 0 || d <= 0)
        return hipErrorInvalidValue;
    if (d > kMaxHeadDim) return hipErrorNotSupported;
    if (d % 8 != 0) return hipErrorInvalidValue;
    out.data = const_cast<std::uint8_t*>(data);
    out.pages = pages;
    out.page_size = page_size;
    out.kv_heads = kv_heads;
    out.groups = cache_groups(d);
    out.head_bytes = static_cast<std::int64_t>(page_size / kCacheKeys) * cache_block_bytes(out.groups);
    // pages * page_bytes has to fit 63 bits: page_bytes under 2^32 does.
    if (out.head_bytes > 0xffffffffLL / kv_heads) return hipErrorInvalidValue;
    out.page_bytes = out.head_bytes * kv_heads;
    return hipSuccess;
}

// -------------------------------------------------------------- wave helpers

// Inclusive prefix sum over the lanes: DPP steps inside rows of 16 lanes, then the last
// lane of each row added to the rows after it.
__device__ __forceinline__ unsigned prefix_sum(unsigned x) {
    int v = static_cast<int>(x);
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2 and 3
    return static_cast<unsigned>(v);
}

// ------------------------------------------------------------- bf16 helpers

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));

// Two floats rounded to nearest even to fp16 or bf16, the first in the low half.
template <bool kBf16>
__device__ __forceinline__ std::uint32_t pack_pair(float a, float b) {
    const float2v x{a, b};
    if constexpr (kBf16)
        return __builtin_bit_cast(std::uint32_t, __builtin_convertvector(x, bf2v));
    else
        return __builtin_bit_cast(std::uint32_t, __builtin_convertvector(x, half2v));
}

// The float that the low (kHalf = 0) or high half of a pair holds.
template <bool kBf16, int kHalf>
__device__ __forceinline__ float half_of(std::uint32_t pair) {
    if constexpr (kBf16)
        return __builtin_bit_cast(float, kHalf ? pair & 0xffff0000u : pair << 16);
    else
        return half_bits_to_float(static_cast<std::uint16_t>(pair >> (16 * kHalf)));
}

}  // namespace tilemix
