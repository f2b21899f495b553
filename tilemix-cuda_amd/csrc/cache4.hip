// Writing and reading the paged 4-bit key/value cache (tilemix_cache4_append,
// tilemix_cache4_gather) for gfx950. Both are bound by memory: every input is
// read once and every output written once; the formulas are in
// include/tilemix_capi.h and the layout of a block in serving.h.
//
// A team of lanes - 8 for d <= 64, 16 above - holds one token's row of one head,
// 8 features a lane (16 bytes), so that a rotation's partner features are one more
// 16-byte load that hits the cache (where half the rotated features are a multiple
// of 8; else single values) and a group's extremes are three DPP steps. The teams of
// a wave hold consecutive tokens of the same head: their key codes are one run of
// the block, and their 16-bit pieces of a value row lie side by side, so that a
// store touches 8 bytes of each line instead of 2. The waves of a workgroup take the
// tokens after one another's, for the same reason, and workgroups that share a block of
// the cache run on one XCD (token_group_of): dealt out one by one, eight L2s would each
// read, or write a piece of, the same lines. A wave takes several heads with the
// cosines and sines kept in registers.
//
// 8192 tokens of 32 query and 8 key heads x 128, rotated, out of place: append 37 to 46 us (4.2
// to 5.2 TB/s of 194 MB), gather of the same rows 10.4 (33.6 MB written, 9.4 read); 16384 rows
// gathered 16.4 to 18. Of a few tokens both are latency: 4 and 3 us.

#include "serving.h"
#include "tilemix_capi.h"

#include <algorithm>
#include <type_traits>

namespace tilemix {
namespace {

constexpr int kCacheThreads = 256;
constexpr int kCacheWaves = kCacheThreads / kWave;
constexpr int kXcds = 8;

struct TokenRows {
    const std::uint16_t* in;
    std::uint16_t* out;
    Rows in_rows, out_rows;
};

struct AppendParams {
    TokenRows q, k, v;
    const float* cos_sin;
    const std::int32_t* token_positions;
    const std::int64_t* slots;
    Cache cache;
    int tokens, positions;
    int q_heads, kv_heads;
    int d, rotary, half;
    int heads_per_wave;
};

struct GatherParams {
    TokenRows k, v;
    const std::int64_t* slots;
    Cache cache;
    int tokens;
    int kv_heads;
    int d;
    int heads_per_wave;
};

// Minimum / maximum / sum over the 8 lanes of a group (DPP steps inside rows of 16 lanes).
template <typename F>
__device__ __forceinline__ float over_8_lanes(float x, F&& f) {
    auto step = [&](auto control) {
        constexpr int kControl = decltype(control)::value;
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kControl, 0xf, 0xf, false));
    };
    x = f(x, step(std::integral_constant<int, 0xb1>{}));   // lane ^ 1
    x = f(x, step(std::integral_constant<int, 0x4e>{}));   // lane ^ 2
    return f(x, step(std::integral_constant<int, 0x141>{}));  // mirrored within 8
}

// Token group (the tokens of a wave) of wave `wave` of workgroup `x` of `count`, a multiple
// of 8: workgroups are dealt round-robin to the 8 XCDs, each of which takes a run.
__device__ __forceinline__ int token_group_of(int x, int count, int wave) {
    return (x % kXcds * (count / kXcds) + x / kXcds) * kCacheWaves + wave;
}

// Where the cache has a slot: byte offset of head 0's block and the token's number in it.
struct Place {
    std::int64_t block;
    int t;
    bool ok;
};
__device__ __forceinline__ Place place_of(const Cache& cache, std::int64_t slot) {
    Place at;
    at.ok = slot >= 0 && slot < cache.pages * cache.page_size;
    const std::int64_t page = at.ok ? slot / cache.page_size : 0;
    const int inside = at.ok ? static_cast<int>(slot - page * cache.page_size) : 0;
    at.block = cache_block_at(page, cache.page_bytes, inside / kCacheKeys, cache_block_bytes(cache.groups));
    at.t = inside % kCacheKeys;
    return at;
}

// Product rounded to fp32 before anything is added to it: the compiler would
// contract it into an fma, and the rotated values, hence the codes, would depend on which.
__device__ __forceinline__ float rounded_product(float a, float b) {
    float product = a * b;
    asm("" : "+v"(product));
    return product;
}

template <bool kBf16>
__device__ __forceinline__ void unpack8(uint4v raw, float (&x)[8]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        x[2 * w] = half_of<kBf16, 0>(raw[w]);
        x[2 * w + 1] = half_of<kBf16, 1>(raw[w]);
    }
}
template <bool kBf16>
__device__ __forceinline__ uint4v pack8(const float (&x)[8]) {
    return uint4v{pack_pair<kBf16>(x[0], x[1]), pack_pair<kBf16>(x[2], x[3]), pack_pair<kBf16>(x[4], x[5]),
                  pack_pair<kBf16>(x[6], x[7])};
}

// How features are turned: not at all; with the feature half the turned ones away, in
// 16-byte pieces or one by one; with their neighbours.
enum class Turn { kNone, kHalves, kHalvesSingle, kPairs };
enum class Kind { kQuery, kKey, kValue };

template <int kGroups, bool kBf16, Turn kTurn>
__global__ __launch_bounds__(kCacheThreads) void cache4_append_kernel(const AppendParams p) {
    constexpr int kTeam = 8 * kGroups;
    constexpr int kTokens = kWave / kTeam;  // of a wave
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int token = token_group_of(blockIdx.x, gridDim.x, wave) * kTokens + lane / kTeam;
    const int chunk = lane % kTeam;  // of 8 features
    const int f0 = 8 * chunk;
    const int first = blockIdx.y * p.heads_per_wave;
    const int last = min(first + p.heads_per_wave, p.q_heads + 2 * p.kv_heads);

    bool valid = token < p.tokens;  // and its position is in the table
    Place at{0, 0, false};
    float cosine[8], sine[8];  // per feature: y = x cosine + partner sine, the sign in the sine
    const bool turned = kTurn != Turn::kNone && f0 < p.rotary;
    const bool second_half = f0 >= p.half;  // (kHalves)
    const int partner = second_half ? f0 - p.half : f0 + p.half;
    if (valid) {
        at = place_of(p.cache, p.slots[token]);
        if constexpr (kTurn != Turn::kNone) {
            const int position = p.token_positions[token];
            valid = position >= 0 && position < p.positions;
            const float* const row = p.cos_sin + static_cast<std::int64_t>(valid ? position : 0) * p.rotary;
            if constexpr (kTurn == Turn::kHalves) {
                if (turned) {
                    const float* const from = row + (second_half ? partner : f0);
                    const float flip = second_half ? 1.0f : -1.0f;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float4v c = *reinterpret_cast<const float4v*>(from + 4 * x);
                        const float4v s = *reinterpret_cast<const float4v*>(from + p.half + 4 * x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) cosine[4 * x + e] = c[e], sine[4 * x + e] = s[e] * flip;
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int f = f0 + e;
                    cosine[e] = 1.0f, sine[e] = 0.0f;
                    if (f < p.rotary) {
                        const bool second = kTurn == Turn::kPairs ? f & 1 : f >= p.half;
                        const int angle = kTurn == Turn::kPairs ? f >> 1 : second ? f - p.half : f;
                        cosine[e] = row[angle];
                        sine[e] = second ? row[p.half + angle] : -row[p.half + angle];
                    }
                }
            }
        }
    }
    const bool live = valid && f0 < p.d;  // holds values
    const bool cached = valid && at.ok;   // writes to the cache, code 0 past d
    const int place = cache_place(at.t);
    std::uint8_t* const head0_block = p.cache.data + at.block;

    // Rows from .. to - 1 of one kind, kBatch of them loaded before the first is taken.
    auto rows_of = [&](auto kind, const TokenRows& rows, int from, int to) __attribute__((always_inline)) {
        constexpr Kind kKind = decltype(kind)::value;
        constexpr bool kTurned = kTurn != Turn::kNone && kKind != Kind::kValue;
        constexpr int kBatch = 4;
        const std::uint16_t* const in = rows.in + token * rows.in_rows.row + f0;
        std::uint16_t* const out = rows.out + token * rows.out_rows.row + f0;
        for (int head = from; head < to; head += kBatch) {
            uint4v own[kBatch], other[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                own[b] = other[b] = uint4v{0u, 0u, 0u, 0u};
                if (live && head + b < to) {
                    const std::uint16_t* const x = in + (head + b) * rows.in_rows.head;
                    own[b] = *reinterpret_cast<const uint4v*>(x);
                    if constexpr (kTurned && kTurn == Turn::kHalves)
                        if (turned) other[b] = *reinterpret_cast<const uint4v*>(x + (partner - f0));
                }
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (head + b >= to) break;
                float x[8];
                unpack8<kBf16>(own[b], x);
                if constexpr (kTurned) {
                    float partners[8];
                    if constexpr (kTurn == Turn::kHalves) {
                        unpack8<kBf16>(other[b], partners);
                    } else if constexpr (kTurn == Turn::kPairs) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) partners[e] = x[e ^ 1];
                    } else {
                        const std::uint16_t* const row = in + (head + b) * rows.in_rows.head - f0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int f = f0 + e;
                            partners[e] = live && f < p.rotary ? half_of<kBf16, 0>(row[f < p.half ? f + p.half : f - p.half]) : 0.0f;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (kTurn == Turn::kHalves ? turned : f0 + e < p.rotary)
                            x[e] = rounded_product(x[e], cosine[e]) + rounded_product(partners[e], sine[e]);
                }
                if (kKind != Kind::kValue && rows.out && live)
                    *reinterpret_cast<uint4v*>(out + (head + b) * rows.out_rows.head) = pack8<kBf16>(x);
                if constexpr (kKind == Kind::kQuery) continue;
                // Extremes of the group; `zero` becomes NaN with any value that is not finite.
                float low = live ? x[0] : INFINITY, high = live ? x[0] : -INFINITY, zero = live ? x[0] * 0.0f : 0.0f;
                if (live) {
#pragma unroll
                    for (int e = 1; e < 8; ++e) {
                        low = fminf(low, x[e]);
                        high = fmaxf(high, x[e]);
                        zero = __builtin_fmaf(x[e], 0.0f, zero);
                    }
                }
                low = over_8_lanes(low, [](float a, float b) { return fminf(a, b); });
                high = over_8_lanes(high, [](float a, float b) { return fmaxf(a, b); });
                zero = over_8_lanes(zero, [](float a, float b) { return a + b; });
                const float minimum = half_of<true, 1>(pack_pair<true>(0.0f, low)) + 0.0f;  // a zero without its sign
                std::uint32_t params = pack_pair<true>((high - minimum) / 15.0f, minimum);
                const float scale = half_of<true, 0>(params);
                const bool finite = zero == 0.0f && fabsf(scale) < INFINITY;  // (-inf: of a minimum past bf16's values)
                const bool coded = finite && scale >= kLeastScale;
                if (!finite) params = 0x7fc07fc0u;
                else if (!coded) params &= 0xffff0000u;
                const float recip = 1.0f / scale;
                std::uint32_t code[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    code[e] = static_cast<std::uint32_t>(
                        __builtin_amdgcn_fmed3f(__builtin_rintf(quotient(x[e] - minimum, scale, recip)), 0.0f, 15.0f));
                const bool written = coded && live;
                if (cached) {
                    std::uint8_t* const block = head0_block + (head + b) * p.cache.head_bytes;
                    if constexpr (kKind == Kind::kKey) {
                        std::uint32_t word = 0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) word |= code[e] << (4 * (e / 2) + 16 * (e % 2));
                        const int m = chunk >> 3, g = (chunk >> 1) & 3, w = chunk & 1;
                        reinterpret_cast<std::uint32_t*>(block)[8 * kGroups * at.t + 2 * kGroups * g + 2 * m + w] = written ? word : 0u;
                    } else {
                        auto* const quarters = reinterpret_cast<std::uint16_t*>(block + cache_values_at(kGroups)) + place;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const std::uint32_t word = code[4 * half] | (code[4 * half + 1] << 4) | (code[4 * half + 2] << 8) |
                                                       (code[4 * half + 3] << 12);
                            quarters[(2 * chunk + half) * kCacheKeys] = static_cast<std::uint16_t>(written ? word : 0u);
                        }
                    }
                    if ((chunk & 7) == 0)
                        reinterpret_cast<std::uint32_t*>(
                            block + (kKind == Kind::kKey ? cache_key_params_at(kGroups) : cache_value_params_at(kGroups)))
                            [(chunk >> 3) * kCacheKeys + place] = params;
                }
            }
        }
    };
    using Query = std::integral_constant<Kind, Kind::kQuery>;
    using Key = std::integral_constant<Kind, Kind::kKey>;
    using Value = std::integral_constant<Kind, Kind::kValue>;
    const int keys = p.q_heads, values = keys + p.kv_heads;  // queries, then keys, then values
    rows_of(Query{}, p.q, first, min(last, keys));
    rows_of(Key{}, p.k, max(first - keys, 0), min(last, values) - keys);
    rows_of(Value{}, p.v, max(first - values, 0), last - values);
}

template <int kGroups, bool kBf16>
__global__ __launch_bounds__(kCacheThreads) void cache4_gather_kernel(const GatherParams p) {
    constexpr int kTeam = 8 * kGroups;
    constexpr int kTokens = kWave / kTeam;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int token = token_group_of(blockIdx.x, gridDim.x, wave) * kTokens + lane / kTeam;
    const int chunk = lane % kTeam, f0 = 8 * chunk;
    if (token >= p.tokens || f0 >= p.d) return;
    const Place at = place_of(p.cache, p.slots[token]);
    if (!at.ok) return;
    const int place = cache_place(at.t);
    const int m = chunk >> 3, g = (chunk >> 1) & 3, w = chunk & 1;
    const int keys = p.k.out ? p.kv_heads : 0, heads = keys + (p.v.out ? p.kv_heads : 0);
    const int first = blockIdx.y * p.heads_per_wave;
    const int last = min(first + p.heads_per_wave, heads);
    const std::uint8_t* const head0_block = p.cache.data + at.block;
    auto rows_of = [&](auto kind, const TokenRows& rows, int from, int to) __attribute__((always_inline)) {
        constexpr bool kKey = decltype(kind)::value == Kind::kKey;
        constexpr int kBatch = 4;
        std::uint16_t* const out = rows.out + token * rows.out_rows.row + f0;
        for (int head = from; head < to; head += kBatch) {
            std::uint32_t params[kBatch], codes[kBatch][2];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const std::uint8_t* const block = head0_block + min(head + b, to - 1) * p.cache.head_bytes;
                params[b] = reinterpret_cast<const std::uint32_t*>(
                    block + (kKey ? cache_key_params_at(kGroups) : cache_value_params_at(kGroups)))[m * kCacheKeys + place];
                if constexpr (kKey) {
                    codes[b][0] = reinterpret_cast<const std::uint32_t*>(block)[8 * kGroups * at.t + 2 * kGroups * g + 2 * m + w];
                } else {
                    const auto* const quarters = reinterpret_cast<const std::uint16_t*>(block + cache_values_at(kGroups)) + place;
#pragma unroll
                    for (int half = 0; half < 2; ++half) codes[b][half] = quarters[(2 * chunk + half) * kCacheKeys];
                }
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (head + b >= to) break;
                const float scale = half_of<true, 0>(params[b]), minimum = half_of<true, 1>(params[b]);
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const std::uint32_t code = kKey ? codes[b][0] >> (4 * (e / 2) + 16 * (e % 2)) : codes[b][e / 4] >> (4 * (e % 4));
                    x[e] = __builtin_fmaf(scale, static_cast<float>(code & 15u), minimum);
                }
                *reinterpret_cast<uint4v*>(out + (head + b) * rows.out_rows.head) = pack8<kBf16>(x);
            }
        }
    };
    rows_of(std::integral_constant<Kind, Kind::kKey>{}, p.k, first, min(last, keys));
    rows_of(std::integral_constant<Kind, Kind::kValue>{}, p.v, max(first - keys, 0), last - keys);
}

// Heads that one wave takes in turn, and the grid: enough waves to fill the device. Less than
// 2^32 threads along a side, which is also what keeps token numbers in 32 bits.
hipError_t plan_rows(int tokens, int groups, std::int64_t heads, int& heads_per_wave, dim3& grid) {
    constexpr int kWavesWanted = 4096;  // (append and gather of 8192 tokens: 1024 62 us, 4096 58, 16384 67)
    const std::int64_t token_groups = (tokens - 1) / (kWave / (8 * groups)) + 1;
    heads_per_wave = static_cast<int>(std::clamp<std::int64_t>(token_groups * heads / kWavesWanted, 1, heads));
    const std::int64_t workgroups = ((token_groups - 1) / kCacheWaves + kXcds) / kXcds * kXcds;
    if (workgroups > 0xffffffffLL / kCacheThreads) return hipErrorInvalidConfiguration;
    grid = dim3(static_cast<unsigned>(workgroups), static_cast<unsigned>((heads - 1) / heads_per_wave + 1));  // y < 2 kWavesWanted
    return hipSuccess;
}

template <int kGroups, Turn kTurn>
hipError_t launch_append(const AppendParams& p, dim3 grid, bool bf16, hipStream_t stream) {
    if (bf16)
        cache4_append_kernel<kGroups, true, kTurn><<<grid, kCacheThreads, 0, stream>>>(p);
    else
        cache4_append_kernel<kGroups, false, kTurn><<<grid, kCacheThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <Turn kTurn>
hipError_t launch_append(const AppendParams& p, dim3 grid, bool bf16, hipStream_t stream) {
    return p.cache.groups == 1 ? launch_append<1, kTurn>(p, grid, bf16, stream) : launch_append<2, kTurn>(p, grid, bf16, stream);
}

template <int kGroups>
hipError_t launch_gather(const GatherParams& p, dim3 grid, bool bf16, hipStream_t stream) {
    if (bf16)
        cache4_gather_kernel<kGroups, true><<<grid, kCacheThreads, 0, stream>>>(p);
    else
        cache4_gather_kernel<kGroups, false><<<grid, kCacheThreads, 0, stream>>>(p);
    return hipGetLastError();
}

// Rows written over what they are computed from have to be the same rows.
bool in_place_ok(const TokenRows& rows) {
    return rows.in != rows.out || (rows.in_rows.row == rows.out_rows.row && rows.in_rows.head == rows.out_rows.head);
}

bool dtype_ok(int dtype) { return dtype == TILEMIX_DTYPE_F16 || dtype == TILEMIX_DTYPE_BF16; }

}  // namespace
}  // namespace tilemix

extern "C" std::size_t tilemix_cache4_block_bytes(int d) {
    if (d <= 0 || d > tilemix::kMaxHeadDim || d % 8 != 0) return 0;
    return static_cast<std::size_t>(tilemix::cache_block_bytes(tilemix::cache_groups(d)));
}

extern "C" std::size_t tilemix_cache4_bytes(std::int64_t pages, int page_size, int kv_heads, int d) {
    alignas(16) static const std::uint8_t any[16] = {};  // an address that passes the check
    tilemix::Cache cache;
    if (tilemix::make_cache(cache, any, pages, page_size, kv_heads, d) != hipSuccess) return 0;
    return static_cast<std::size_t>(cache.pages) * static_cast<std::size_t>(cache.page_bytes);
}

extern "C" int tilemix_cache4_append(const TileMixCache4AppendArgs* args, void* stream) {
    using namespace tilemix;
    if (!args) return hipErrorInvalidValue;
    const TileMixCache4AppendArgs& a = *args;
    AppendParams p{};
    const hipError_t cache_ok = make_cache(p.cache, a.cache, a.pages, a.page_size, a.kv_heads, a.d);
    if (cache_ok != hipSuccess) return cache_ok;
    if (a.tokens < 0 || !dtype_ok(a.dtype) || a.rotary_dim < 0 || a.rotary_dim > a.d || a.rotary_dim % 2 != 0 ||
        (a.Q && a.q_heads <= 0) || (!a.Q) != (!a.Q_out) ||
        (a.rotary_dim > 0 && (a.positions <= 0 || !a.cos_sin || !a.token_positions)))
        return hipErrorInvalidValue;
    p.q_heads = a.Q ? a.q_heads : 0;
    if (p.q_heads > 0x3fffffff || a.kv_heads > 0x1fffffff) return hipErrorInvalidValue;
    p.q.in = a.Q, p.q.out = a.Q_out;
    p.k.in = a.K, p.k.out = a.K_out;
    p.v.in = a.V, p.v.out = nullptr;
    if ((a.Q && (!make_rows(p.q.in_rows, a.Q, a.tokens, a.q_heads, a.d, a.q_row_stride, a.q_head_stride, 8) ||
                 !make_rows(p.q.out_rows, a.Q_out, a.tokens, a.q_heads, a.d, a.q_out_row_stride, a.q_out_head_stride, 8))) ||
        !make_rows(p.k.in_rows, a.K, a.tokens, a.kv_heads, a.d, a.k_row_stride, a.k_head_stride, 8) ||
        (a.K_out && !make_rows(p.k.out_rows, a.K_out, a.tokens, a.kv_heads, a.d, a.k_out_row_stride, a.k_out_head_stride, 8)) ||
        !make_rows(p.v.in_rows, a.V, a.tokens, a.kv_heads, a.d, a.v_row_stride, a.v_head_stride, 8))
        return hipErrorInvalidValue;
    if (a.tokens == 0) return hipSuccess;
    if (!a.slots || (a.Q && !in_place_ok(p.q)) || !in_place_ok(p.k)) return hipErrorInvalidValue;
    dim3 grid;
    const hipError_t planned =
        plan_rows(a.tokens, p.cache.groups, p.q_heads + std::int64_t{2} * a.kv_heads, p.heads_per_wave, grid);
    if (planned != hipSuccess) return planned;
    p.cos_sin = a.cos_sin;
    p.token_positions = a.token_positions;
    p.slots = a.slots;
    p.tokens = a.tokens;
    p.positions = a.positions;
    p.kv_heads = a.kv_heads;
    p.d = a.d;
    p.rotary = a.rotary_dim;
    p.half = a.rotary_dim / 2;
    const hipError_t found = check_device();
    if (found != hipSuccess) return found;
    const bool bf16 = a.dtype == TILEMIX_DTYPE_BF16;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.rotary == 0) return launch_append<Turn::kNone>(p, grid, bf16, s);
    if (a.interleaved) return launch_append<Turn::kPairs>(p, grid, bf16, s);
    const bool pieces = p.half % 8 == 0 && reinterpret_cast<std::uintptr_t>(p.cos_sin) % 16 == 0;
    return pieces ? launch_append<Turn::kHalves>(p, grid, bf16, s) : launch_append<Turn::kHalvesSingle>(p, grid, bf16, s);
}

extern "C" int tilemix_cache4_gather(const TileMixCache4GatherArgs* args, void* stream) {
    using namespace tilemix;
    if (!args) return hipErrorInvalidValue;
    const TileMixCache4GatherArgs& a = *args;
    GatherParams p{};
    const hipError_t cache_ok = make_cache(p.cache, a.cache, a.pages, a.page_size, a.kv_heads, a.d);
    if (cache_ok != hipSuccess) return cache_ok;
    if (a.tokens < 0 || !dtype_ok(a.dtype) || a.kv_heads > 0x1fffffff) return hipErrorInvalidValue;
    if (a.tokens == 0) return hipSuccess;
    if (!a.slots || (!a.K_out && !a.V_out)) return hipErrorInvalidValue;
    p.k.out = a.K_out;
    p.v.out = a.V_out;
    if ((a.K_out && !make_rows(p.k.out_rows, a.K_out, a.tokens, a.kv_heads, a.d, a.k_row_stride, a.k_head_stride, 8)) ||
        (a.V_out && !make_rows(p.v.out_rows, a.V_out, a.tokens, a.kv_heads, a.d, a.v_row_stride, a.v_head_stride, 8)))
        return hipErrorInvalidValue;
    p.slots = a.slots;
    p.tokens = a.tokens;
    p.kv_heads = a.kv_heads;
    p.d = a.d;
    dim3 grid;
    const hipError_t planned =
        plan_rows(a.tokens, p.cache.groups, std::int64_t{a.kv_heads} * ((a.K_out ? 1 : 0) + (a.V_out ? 1 : 0)), p.heads_per_wave, grid);
    if (planned != hipSuccess) return planned;
    const hipError_t found = check_device();
    if (found != hipSuccess) return found;
    const bool bf16 = a.dtype == TILEMIX_DTYPE_BF16;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return p.cache.groups == 1 ? launch_gather<1>(p, grid, bf16, s) : launch_gather<2>(p, grid, bf16, s);
}
