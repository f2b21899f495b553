// One decode step over the paged 4-bit cache for gfx950 (tilemix_attention_cache4):
// the rows of a key head's query heads against all cached tokens of a sequence.
//
// With x = minimum + scale * code per group of 64 features,
//   q . k = sum_m scale_m (sum_f code_f q_f) + minimum_m (sum_f q_f)
//   sum_t p_t v_t = sum_t code_t (p_t scale_t) + sum_t p_t minimum_t,
// so codes enter the matrix cores as they are: 16 + code is exact in fp16 and bf16
// and its bits are the code's, shifted, under a constant exponent - one shift and
// one and-or for two codes, no subtraction, no scaling. The 16 is taken out by the
// accumulator's start (-16 sum q) and beside the minimum. q . k is exact but for
// fp32 sums; of p scale, two bf16 parts (hi + lo, 2^-17 of it) are multiplied, as
// bf16 holds any scale (fp16 would not).
//
// What bounds it is memory: 144 bytes a token and head at d = 128. The cache lies
// in blocks of 32 tokens in the order of these operands (serving.h): a wave takes
// a block per step, each load of a wave one contiguous KiB (parameters: 128 bytes
// read by all), the next block's loads issued before a block is computed.
//
// Split of the work: the blocks of all sequences and heads are dealt out in parts
// of equal length, found on the device from the lengths (plan): lengths differ, and
// the host does not know them. The parts of one sequence and head meet in the
// workspace, where the workgroup that arrives last merges them in order.

#include "attention_common.h"
#include "serving.h"
#include "tilemix_capi.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace tilemix {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kTileRows = 16;     // query rows of a workgroup
constexpr int kPartsWanted = 512;  // two workgroups per CU
constexpr int kLeastSteps = 8;     // blocks of a part: two for each wave
// Parts of sequences and heads that have several: n of them cover more than n - 1
// times a part's length, so there are fewer than kPartsWanted beside each one's first.
constexpr int kPartsKept = 2 * kPartsWanted;
constexpr int kPartFloats = kTileRows * (kMaxHeadDim + 2);
constexpr std::size_t kWorkspaceBytes = kPartsKept * sizeof(unsigned) + std::size_t{kPartsKept} * kPartFloats * sizeof(float);

struct DecodeParams {
    const std::uint16_t* Q;
    std::uint16_t* O;
    Cache cache;
    const std::int32_t* table;
    const std::int32_t* lengths;
    unsigned* arrivals;  // [kPartsKept], zero between calls
    float* parts;
    Rows q, o;
    std::int64_t table_stride;
    int batch;
    int group;  // query heads per key head
    int tiles;  // of kTileRows query heads per key head
    int d;
    int most_tokens;  // max_pages * page_size
    int negate;
    float score_log2;
};

typedef __amdgpu_buffer_rsrc_t Rsrc;

template <bool kBf16>
__device__ __forceinline__ float4v mfma_16x16x32(uint4v a, uint4v b, float4v c) {
    if constexpr (kBf16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// 16 + code of the nibbles j of a word's halves, as a pair of fp16 (mantissa bits
// 9 .. 6 under exponent 4) or bf16 (bits 6 .. 3): two instructions, the second
// written out, as the compiler, given two constants, makes it an and and an or.
template <bool kBf16>
struct Codes {
    std::uint32_t mask;  // in a vector register: an instruction takes one scalar
    __device__ __forceinline__ Codes() {
        if constexpr (kBf16) asm("v_mov_b32 %0, 0x00780078" : "=v"(mask));
        else asm("v_mov_b32 %0, 0x03c003c0" : "=v"(mask));
    }
    template <int j>
    __device__ __forceinline__ std::uint32_t pair(std::uint32_t word) const {
        constexpr int kUp = (kBf16 ? 3 : 6) - 4 * j;
        const std::uint32_t shifted = kUp >= 0 ? word << (kUp & 31) : word >> (-kUp & 31);
        std::uint32_t out;
        asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(out) : "v"(shifted), "v"(mask), "s"(kBf16 ? 0x41804180u : 0x4c004c00u));
        return out;
    }
    __device__ __forceinline__ uint4v all(std::uint32_t word) const {  // the word's 8 codes
        return uint4v{pair<0>(word), pair<1>(word), pair<2>(word), pair<3>(word)};
    }
    template <int j>
    __device__ __forceinline__ uint4v of(uint4v words) const {  // nibbles j of four words
        return uint4v{pair<j>(words[0]), pair<j>(words[1]), pair<j>(words[2]), pair<j>(words[3])};
    }
};

// Sum / maximum over the four lanes r, r + 16, r + 32, r + 48, in each of them.
__device__ __forceinline__ void permlane16_swap(float& a, float& b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ float groups_max(float x) {
    float a = x, b = x;
    permlane16_swap(a, b);
    a = fmaxf(a, b);
    b = a;
    permlane32_swap(a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float groups_sum(float x) {
    float a = x, b = x;
    permlane16_swap(a, b);
    a = a + b;
    b = a;
    permlane32_swap(a, b);
    return a + b;
}

__device__ __forceinline__ int prefix_sum(int v, int lane) {  // inclusive, over the lanes
#pragma unroll
    for (int step = 1; step < kWave; step <<= 1) {
        const int other = __shfl_up(v, step);
        if (lane >= step) v += other;
    }
    return v;
}

// A workgroup's part: blocks first .. end - 1 of a sequence, head and row tile.
struct Part {
    int sequence, length, head, tile;
    int first, end;
    int index, count;  // of the sequence and head's parts
    int kept;          // workspace place of its part 0 (count > 1)
};

__device__ __forceinline__ int blocks_of(const DecodeParams& p, int b) {
    return b < p.batch ? (min(max(p.lengths[b], 0), p.most_tokens) + kCacheKeys - 1) / kCacheKeys : 0;
}

// Part number `number` of the call; false past the last. Wave-uniform.
__device__ __forceinline__ bool plan(const DecodeParams& p, int number, int lane, Part& part) {
    const int heads = p.cache.kv_heads * p.tiles;
    std::int64_t blocks = 0;
    for (int b = lane; b < p.batch; b += kWave) blocks += blocks_of(p, b);
#pragma unroll
    for (int step = kWave / 2; step > 0; step >>= 1) blocks += __shfl_xor(blocks, step);
    // (A sequence has under 2^26 blocks: longer parts make no difference.)
    const std::int64_t wanted = min((blocks * heads + kPartsWanted - 1) / kPartsWanted, std::int64_t{1} << 26);
    const int length = __builtin_amdgcn_readfirstlane(max(static_cast<int>(wanted), kLeastSteps));
    const int parts_wanted = number / heads;  // parts of whole sequences before this one's
    int parts_before = 0, kept_before = 0;
    for (int base = 0; base < p.batch; base += kWave) {
        const int b = base + lane;
        const int mine = blocks_of(p, b);
        const int count = b < p.batch ? max((mine + length - 1) / length, 1) : 0;
        const int parts = prefix_sum(count, lane) + parts_before;
        const int kept = prefix_sum(count > 1 ? count : 0, lane) + kept_before;
        const std::uint64_t past = __ballot(parts > parts_wanted);
        if (past) {
            const int at = __builtin_ctzll(past);
            part.sequence = base + at;
            part.count = __builtin_amdgcn_readlane(count, at);
            part.index = parts_wanted - (__builtin_amdgcn_readlane(parts, at) - part.count);
            const int in_sequence = number % heads;
            part.head = in_sequence / p.tiles;
            part.tile = in_sequence - part.head * p.tiles;
            const int total = __builtin_amdgcn_readlane(mine, at);
            part.first = min(part.index * length, total);
            part.end = min(part.first + length, total);
            part.kept = (__builtin_amdgcn_readlane(kept, at) - part.count) * heads + in_sequence * part.count;
            part.length = min(max(p.lengths[part.sequence], 0), p.most_tokens);
            return true;
        }
        parts_before = __builtin_amdgcn_readlane(parts, kWave - 1);
        kept_before = __builtin_amdgcn_readlane(kept, kWave - 1);
    }
    return false;
}

// A block as loaded: 16 (two groups of features) or 8 bytes of codes per lane and
// 16 tokens / group, and the parameters of the lane's 8 tokens.
template <int kGroups>
struct Block {
    std::uint32_t k[2][2 * kGroups];
    uint4v v[kGroups];
    uint4v k_params[kGroups][2], v_params[kGroups][2];
    std::uint32_t row_params[2][kGroups];  // of token 16 b + r
};

template <int kGroups, bool kBf16>
__global__ __launch_bounds__(kThreads, 2) void cache4_attention_kernel(const DecodeParams p) {
    constexpr int kDP = 64 * kGroups;
    constexpr int kFeatures = 4 * kGroups;  // of a thread in the merges
    __shared__ __attribute__((aligned(16))) float lds_o[kWaves][kTileRows][kDP];
    __shared__ float lds_ml[kWaves][kTileRows][2];
    __shared__ int lds_last;

    const int tid = threadIdx.x;
    const int lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15;  // token of a score block / feature quarter (A operands), query row (B operands, results)
    const int g = lane >> 4;
    Part part;
    if (!plan(p, blockIdx.x, lane, part)) return;
    const int rows = min(p.group - part.tile * kTileRows, kTileRows);
    const int head0 = part.head * p.group + part.tile * kTileRows;
    const int d = p.d;

    // ------------------------------------------------------------ pages
    // Lane l of the window holds page number window + l of the sequence.
    const int per_page = p.cache.page_size / kCacheKeys;
    const std::int32_t* const table = p.table + part.sequence * p.table_stride;
    const int pages = (part.length + p.cache.page_size - 1) / p.cache.page_size;
    int page = (part.first + wave) / per_page, inside = (part.first + wave) - page * per_page;
    int window = page;
    int window_page = 0;
    auto load_window = [&]() __attribute__((always_inline)) { window_page = window + lane < pages ? table[window + lane] : -1; };
    load_window();
    const std::uint8_t* const head_data = p.cache.data + part.head * p.cache.head_bytes;
    constexpr int kBlockBytes = cache_block_bytes(kGroups);
    // The block of `step` (page and inside), or null where its page is no page of the cache.
    auto block_at = [&]() __attribute__((always_inline)) {
        if (page - window >= kWave) {
            window = page;
            load_window();
        }
        const int number = __builtin_amdgcn_readlane(window_page, page - window);
        return number >= 0 && number < p.cache.pages ? head_data + number * p.cache.page_bytes + inside * kBlockBytes : nullptr;
    };
    auto advance = [&]() __attribute__((always_inline)) {
        inside += kWaves;
        while (inside >= per_page) {
            inside -= per_page;
            ++page;
        }
    };
    auto load = [&](Block<kGroups>& block, const std::uint8_t* data) __attribute__((always_inline)) {
        const Rsrc rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<std::uint8_t*>(data), 0, kBlockBytes, kBufferFlags);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int at = 32 * kGroups * (16 * b + r) + 8 * kGroups * g;
            if constexpr (kGroups == 2) {
                const uint4v words = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
#pragma unroll
                for (int w = 0; w < 4; ++w) block.k[b][w] = words[w];
            } else {
                const uint2v words = __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0);
                block.k[b][0] = words[0];
                block.k[b][1] = words[1];
            }
        }
#pragma unroll
        for (int m = 0; m < kGroups; ++m)
            block.v[m] = __builtin_amdgcn_raw_buffer_load_b128(rs, cache_values_at(kGroups) + 64 * (16 * m + r) + 16 * g, 0, 0);
#pragma unroll
        for (int m = 0; m < kGroups; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int at = 128 * m + 32 * g + 16 * x;
                block.k_params[m][x] = __builtin_amdgcn_raw_buffer_load_b128(rs, cache_key_params_at(kGroups) + at, 0, 0);
                block.v_params[m][x] = __builtin_amdgcn_raw_buffer_load_b128(rs, cache_value_params_at(kGroups) + at, 0, 0);
                block.row_params[x][m] = __builtin_amdgcn_raw_buffer_load_b32(
                    rs, cache_key_params_at(kGroups) + 128 * m + 4 * (8 * (r >> 2) + 4 * x + (r & 3)), 0, 0);
            }
    };

    // A wave's blocks: part.first + wave, + kWaves, ... Those without a page are passed over.
    int step = part.first + wave;
    const std::uint8_t* data = nullptr;
    auto find = [&]() __attribute__((always_inline)) {
        for (; step < part.end; step += kWaves, advance()) {
            data = block_at();
            if (data) break;
        }
    };
    Block<kGroups> even, odd;
    find();
    if (step < part.end) load(even, data);

    // ------------------------------------------------------------ Q
    uint4v qf[kGroups][2];
    float q_sum[kGroups];  // of the row's features
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        q_sum[m] = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int feature = 64 * m + 16 * g + 8 * w;
            qf[m][w] = uint4v{0u, 0u, 0u, 0u};
            if (r < rows && feature < d)
                qf[m][w] = *reinterpret_cast<const uint4v*>(p.Q + part.sequence * p.q.row + (head0 + r) * p.q.head + feature);
            if (p.negate) qf[m][w] ^= 0x80008000u;
#pragma unroll
            for (int x = 0; x < 4; ++x) q_sum[m] += half_of<kBf16, 0>(qf[m][w][x]) + half_of<kBf16, 1>(qf[m][w][x]);
        }
        q_sum[m] = groups_sum(q_sum[m]);
    }
    // B operand against (scale, minimum) words: 0, then sum q in three bf16 parts
    // (all of its 24 bits), the first two in the lanes of group 0, the third in those of 1.
    uint4v q_sums{0u, 0u, 0u, 0u};
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        const std::uint32_t first = pack_pair<true>(0.0f, q_sum[m]);
        const float rest = q_sum[m] - half_of<true, 1>(first);
        const std::uint32_t second = pack_pair<true>(0.0f, rest);
        const std::uint32_t third = pack_pair<true>(0.0f, rest - half_of<true, 1>(second));
        q_sums[m] = g == 0 ? first : g == 1 ? third : 0u;
        q_sums[kGroups + m] = g == 0 ? second : 0u;
    }
    const Codes<kBf16> key_codes;
    const Codes<true> value_codes;
    const uint4v ones{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

    float4v o[kGroups][4];  // o[m][f][i]: row r, feature 64 m + 16 g + 4 i + f
    float below[kGroups];     // the lane's part of sum p minimum
    float4v sixteen[kGroups];  // sum p scale, as multiplied, in every element
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        below[m] = 0.0f;
        sixteen[m] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int f = 0; f < 4; ++f) o[m][f] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float row_max = -INFINITY, row_sum = 0.0f;  // row_sum: the lane's part

    auto compute = [&](const Block<kGroups>& block, int at) __attribute__((always_inline)) {
        // Slot e of group g: token 16 (e / 4) + 4 g + e % 4 of the block.
        float4v s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const auto& words = block.row_params[b];
            const uint4v params = kGroups == 2 ? uint4v{words[0], words[kGroups - 1], words[0], words[kGroups - 1]}
                                               : uint4v{words[0], words[0], 0u, 0u};
            s[b] = mfma_16x16x32<true>(params, q_sums, float4v{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int m = 0; m < kGroups; ++m) {
                const float start = -16.0f * q_sum[m];
                float4v acc{start, start, start, start};
#pragma unroll
                for (int w = 0; w < 2; ++w) acc = mfma_16x16x32<kBf16>(key_codes.all(block.k[b][2 * m + w]), qf[m][w], acc);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[b][i] = __builtin_fmaf(half_of<true, 0>(block.k_params[m][b][i]), acc[i], s[b][i]);
            }
        }
        uint4v v_params[kGroups][2];
#pragma unroll
        for (int m = 0; m < kGroups; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) v_params[m][x] = block.v_params[m][x];
        const int left = part.length - at * kCacheKeys;  // tokens from the block's first on
        if (left < kCacheKeys) {
            // Past the length the block may hold anything, NaN included.
            int mine = left - 4 * g;
            asm volatile("" : "+v"(mine));  // a branch: one block in a sequence takes it
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (16 * (e / 4) + e % 4 >= mine) {
                    s[e / 4][e % 4] = -INFINITY;
#pragma unroll
                    for (int m = 0; m < kGroups; ++m) v_params[m][e / 4][e % 4] = 0u;
                }
        }
        const float c = p.score_log2;  // > 0
        const float top = max3(max3(s[0][0], s[0][1], s[0][2]), max3(s[0][3], s[1][0], s[1][1]), max3(s[1][2], s[1][3], s[1][3])) * c;
        if (__any(top > row_max + kLazyRescale)) {
            const float m_new = fmaxf(row_max, groups_max(top));
            const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(row_max - m_new);
            row_max = m_new;
#pragma unroll
            for (int m = 0; m < kGroups; ++m) {
                below[m] *= alpha;
                sixteen[m] *= alpha;
#pragma unroll
                for (int f = 0; f < 4; ++f) o[m][f] *= alpha;
            }
            row_sum *= alpha;
        }
        const float neg_m = row_max == -INFINITY ? 0.0f : -row_max;
        float prob[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            prob[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e / 4][e % 4], c, neg_m));
            row_sum += prob[e];
        }
#pragma unroll
        for (int m = 0; m < kGroups; ++m) {
            uint4v high, low;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float scaled[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int e = 2 * t + x;
                    const std::uint32_t params = v_params[m][e / 4][e % 4];
                    scaled[x] = prob[e] * half_of<true, 0>(params);
                    below[m] = __builtin_fmaf(prob[e], half_of<true, 1>(params), below[m]);
                }
                high[t] = pack_pair<true>(scaled[0], scaled[1]);
                low[t] = pack_pair<true>(scaled[0] - half_of<true, 0>(high[t]), scaled[1] - half_of<true, 1>(high[t]));
            }
            const uint4v a0 = value_codes.template of<0>(block.v[m]), a1 = value_codes.template of<1>(block.v[m]),
                         a2 = value_codes.template of<2>(block.v[m]), a3 = value_codes.template of<3>(block.v[m]);
            for (const uint4v& part_of_p : {high, low}) {
                o[m][0] = mfma_16x16x32<true>(a0, part_of_p, o[m][0]);
                o[m][1] = mfma_16x16x32<true>(a1, part_of_p, o[m][1]);
                o[m][2] = mfma_16x16x32<true>(a2, part_of_p, o[m][2]);
                o[m][3] = mfma_16x16x32<true>(a3, part_of_p, o[m][3]);
                sixteen[m] = mfma_16x16x32<true>(ones, part_of_p, sixteen[m]);
            }
        }
    };
    // Two blocks a turn, each loading the other's before it is computed; every wave
    // leaves when its blocks run out.
    while (step < part.end) {
        const int now = step;
        step += kWaves;
        advance();
        find();
        const int second = step;
        if (second < part.end) load(odd, data);
        compute(even, now);
        if (second >= part.end) break;
        step += kWaves;
        advance();
        find();
        if (step < part.end) load(even, data);
        compute(odd, second);
    }

    // ------------------------------------------------------- merge of waves
    row_sum = groups_sum(row_sum);
    if (g == 0) {
        lds_ml[wave][r][0] = row_max;
        lds_ml[wave][r][1] = row_sum;
    }
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        const float rest = __builtin_fmaf(-16.0f, sixteen[m][0], groups_sum(below[m]));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4v*>(&lds_o[wave][r][64 * m + 16 * g + 4 * i]) =
                float4v{o[m][0][i] + rest, o[m][1][i] + rest, o[m][2][i] + rest, o[m][3][i] + rest};
    }
    __syncthreads();
    const int row = tid >> 4, f0 = kFeatures * (tid & 15);
    float row_m = -INFINITY, row_l = 0.0f;
    float4v acc[kGroups];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) row_m = fmaxf(row_m, lds_ml[w][row][0]);
#pragma unroll
    for (int x = 0; x < kGroups; ++x) acc[x] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        // (A wave whose scores are all NaN has the maximum -inf, and a NaN sum.)
        const float m_w = lds_ml[w][row][0];
        const float weight = m_w == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_w - row_m);
        row_l += weight * lds_ml[w][row][1];
#pragma unroll
        for (int x = 0; x < kGroups; ++x) acc[x] += weight * *reinterpret_cast<const float4v*>(&lds_o[w][row][f0 + 4 * x]);
    }
    const bool mine = row < rows;

    // ------------------------------------------------------- merge of parts
    if (part.count > 1) {
        if (part.kept + part.count > kPartsKept) return;  // never: see kPartsKept
        constexpr int kStride = kTileRows * kDP, kStates = kTileRows * 2;
        float* const states = p.parts + static_cast<std::size_t>(kPartsKept) * kTileRows * kMaxHeadDim;
        const Rsrc ro = shared_rows(p.parts, std::int64_t{kPartsKept} * kTileRows * kMaxHeadDim);
        const Rsrc rml = shared_rows(states, std::int64_t{kPartsKept} * kStates);
        if (mine) {
            const int at = part.kept + part.index;
#pragma unroll
            for (int x = 0; x < kGroups; ++x)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4v, acc[x]), ro,
                                                       (at * kStride + row * kDP + f0 + 4 * x) * 4, 0, kDeviceScope);
            if (f0 == 0)
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uint2v, float2v{row_m, row_l}), rml,
                                                      (at * kStates + 2 * row) * 4, 0, kDeviceScope);
        }
        if (!last_arrival(p.arrivals + part.kept, part.count, &lds_last)) return;
        if (!mine) return;
        row_m = -INFINITY;
        row_l = 0.0f;
#pragma unroll
        for (int x = 0; x < kGroups; ++x) acc[x] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int kBatch = 8;
        for (int s0 = 0; s0 < part.count; s0 += kBatch) {
            float2v state[kBatch];
            float4v value[kBatch][kGroups];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int at = part.kept + min(s0 + u, part.count - 1);
                state[u] = __builtin_bit_cast(
                    float2v, __builtin_amdgcn_raw_buffer_load_b64(rml, (at * kStates + 2 * row) * 4, 0, kDeviceScope));
#pragma unroll
                for (int x = 0; x < kGroups; ++x)
                    value[u][x] = __builtin_bit_cast(
                        float4v, __builtin_amdgcn_raw_buffer_load_b128(ro, (at * kStride + row * kDP + f0 + 4 * x) * 4, 0,
                                                                       kDeviceScope));
            }
            merge_batch<kBatch, true>(
                row_m, row_l, part.count - s0, [&](int u) __attribute__((always_inline)) { return state[u]; },
                [&](int u, PartWeights w) __attribute__((always_inline)) {
#pragma unroll
                    for (int x = 0; x < kGroups; ++x) acc[x] = merged(acc[x], value[u][x], w);
                });
        }
    }
    if (!mine) return;
    const float inverse = row_l == 0.0f ? 0.0f : 1.0f / row_l;  // 0: no token
    std::uint16_t* const out = p.O + part.sequence * p.o.row + (head0 + row) * p.o.head + f0;
#pragma unroll
    for (int x = 0; x < kGroups; ++x)
        if (f0 + 4 * x < d)
            *reinterpret_cast<uint2v*>(out + 4 * x) = uint2v{pack_pair<kBf16>(acc[x][0] * inverse, acc[x][1] * inverse),
                                                             pack_pair<kBf16>(acc[x][2] * inverse, acc[x][3] * inverse)};
}

}  // namespace
}  // namespace tilemix

extern "C" std::size_t tilemix_attention_cache4_workspace_bytes(void) { return tilemix::kWorkspaceBytes; }

extern "C" int tilemix_attention_cache4(const TileMixCache4AttentionArgs* args, void* stream) {
    using namespace tilemix;
    if (!args) return hipErrorInvalidValue;
    const TileMixCache4AttentionArgs& a = *args;
    DecodeParams p{};
    const hipError_t cache_ok = make_cache(p.cache, a.cache, a.pages, a.page_size, a.kv_heads, a.d);
    if (cache_ok != hipSuccess) return cache_ok;
    if (a.batch < 0 || a.q_heads <= 0 || a.q_heads % a.kv_heads != 0 || a.max_pages <= 0 || a.table_stride < 0 ||
        (a.table_stride > 0 && a.table_stride < a.max_pages) || a.table_stride > 0x7fffffffLL ||
        !std::isfinite(a.score_scale) || (a.dtype != TILEMIX_DTYPE_F16 && a.dtype != TILEMIX_DTYPE_BF16) ||
        !make_rows(p.q, a.Q, a.batch, a.q_heads, a.d, a.q_row_stride, a.q_head_stride, 8) ||
        !make_rows(p.o, a.O, a.batch, a.q_heads, a.d, a.o_row_stride, a.o_head_stride, 4))
        return hipErrorInvalidValue;
    if (!a.workspace || !aligned(a.workspace, 16) || a.workspace_bytes < kWorkspaceBytes) return hipErrorInvalidValue;
    if (a.batch == 0) return hipSuccess;
    if (!a.block_table || !a.lengths) return hipErrorInvalidValue;
    p.Q = a.Q;
    p.O = a.O;
    p.table = a.block_table;
    p.lengths = a.lengths;
    p.arrivals = static_cast<unsigned*>(a.workspace);
    p.parts = reinterpret_cast<float*>(p.arrivals + kPartsKept);
    p.table_stride = a.table_stride ? a.table_stride : a.max_pages;
    p.batch = a.batch;
    p.group = a.q_heads / a.kv_heads;
    p.tiles = (p.group - 1) / kTileRows + 1;
    p.d = a.d;
    // A multiple of 32 under 2^31, so that block counts do not overflow.
    p.most_tokens = static_cast<int>(std::min<std::int64_t>(static_cast<std::int64_t>(a.max_pages) * a.page_size, 0x7fffffe0LL));
    p.negate = a.score_scale < 0.0f;
    // (Of a score_scale of 0 the smallest number: a hidden token's -inf times it is still -inf.)
    p.score_log2 = std::max(std::fabs(a.score_scale) * kLog2e, FLT_MIN);
    // The parts wanted, and one more per sequence, head and tile whose last part is not whole.
    const std::int64_t heads = static_cast<std::int64_t>(a.kv_heads) * p.tiles;
    const std::int64_t most = (p.most_tokens / kCacheKeys + kLeastSteps - 1) / kLeastSteps;  // of one of them
    const std::int64_t items = a.batch * heads;
    if (items > 0x3fffffff) return hipErrorInvalidConfiguration;
    const std::int64_t grid = std::min<std::int64_t>(kPartsWanted + items, items * std::max<std::int64_t>(most, 1));
    const hipError_t found = check_device();
    if (found != hipSuccess) return found;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool bf16 = a.dtype == TILEMIX_DTYPE_BF16;
    const unsigned workgroups = static_cast<unsigned>(grid);
    if (p.cache.groups == 1)
        bf16 ? cache4_attention_kernel<1, true><<<workgroups, kThreads, 0, s>>>(p)
             : cache4_attention_kernel<1, false><<<workgroups, kThreads, 0, s>>>(p);
    else
        bf16 ? cache4_attention_kernel<2, true><<<workgroups, kThreads, 0, s>>>(p)
             : cache4_attention_kernel<2, false><<<workgroups, kThreads, 0, s>>>(p);
    return hipGetLastError();
}
