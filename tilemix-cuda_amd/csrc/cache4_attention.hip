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
// a block per step, from a ring of LDS slots of its own that LDS DMA fills in
// contiguous KiB pieces two blocks ahead. (Held in registers, two blocks ahead do not
// fit beside the accumulators, and one ahead leaves waves waiting.)
//
// Split of the work: the blocks of all sequences and heads, one after the other, are
// cut into ranges of equal length, one per workgroup (two or three a CU, one round),
// found on the device from the lengths (first_segment): lengths differ, and the host does not
// know them. A range is a series of segments - blocks of one sequence and head; a
// segment's queries and first blocks are on their way while the one before is merged over
// the waves. Only a range's first and last segment can be a part of a sequence and
// head: those go to the workspace, where the workgroup that arrives last merges them in order.

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
constexpr int kGroupsPerUnit = 2;  // workgroups of a CU that registers are allocated for
constexpr int kSlots = 3;         // blocks in a wave's ring: one computed, two under way
constexpr int kTileRows = 16;     // query rows of a workgroup
constexpr int kLeastSteps = 8;  // blocks of a range: two for each wave
constexpr int kRanges = 512;    // at most: workgroups that the device holds at once
// The workspace: arrival counters, then rows of O and their states for the two parts
// (one continued, one to be continued) that a range can have.
constexpr std::size_t kWorkspaceBytes =
    kRanges * sizeof(unsigned) + std::size_t{2} * kRanges * kTileRows * (kMaxHeadDim + 2) * sizeof(float);

struct DecodeParams {
    const std::uint16_t* Q;
    std::uint16_t* O;
    Cache cache;
    const std::int32_t* table;
    const std::int32_t* lengths;
    unsigned* arrivals;  // [kRanges], zero between calls
    float* part_o;       // [2 kRanges][kTileRows][64 groups]
    float* part_ml;      // [2 kRanges][kTileRows][2]
    int ranges;
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
__device__ __forceinline__ unsigned lane_value(unsigned v, int lane) {
    return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

__device__ __forceinline__ int length_of(const DecodeParams& p, int b) { return min(max(p.lengths[b], 0), p.most_tokens); }
// Blocks of sequence b: under 2^26, so that 64 sequences' fit 32 bits. An empty one counts
// as one block (without a page), so that some range has it and writes its zeros.
__device__ __forceinline__ unsigned blocks_of(const DecodeParams& p, int b) {
    return b < p.batch ? static_cast<unsigned>(max((length_of(p, b) + kCacheKeys - 1) / kCacheKeys, 1)) : 0u;
}

// Blocks first .. end - 1 of a sequence and head (of its `blocks`).
struct Segment {
    int sequence, item;  // item: head * tiles + row tile
    int first, end, blocks;
    int length;               // tokens of the sequence
    std::int64_t start;       // the sequence and head's first block, among all
};

// The length of a range, and the segment in which range number `range` begins; false past
// the last range. Wave-uniform.
__device__ __forceinline__ bool first_segment(const DecodeParams& p, int range, int lane, Segment& segment, std::int64_t& length) {
    const int heads = p.cache.kv_heads * p.tiles;
    const unsigned kept = blocks_of(p, lane);  // of the first kWave sequences
    std::int64_t total = lane_value(prefix_sum(kept), kWave - 1);
    for (int base = kWave; base < p.batch; base += kWave) total += lane_value(prefix_sum(blocks_of(p, base + lane)), kWave - 1);
    total *= heads;
    length = max((total + p.ranges - 1) / p.ranges, std::int64_t{kLeastSteps});
    const std::int64_t begin = range * length;
    if (begin >= total) return false;
    std::int64_t before = 0;  // blocks of one head in the sequences before
    for (int base = 0;; base += kWave) {
        const unsigned mine = base == 0 ? kept : blocks_of(p, base + lane);
        const unsigned sum = prefix_sum(mine);
        const std::uint64_t past = __ballot((before + sum) * heads > begin);
        if (past) {
            const int at = __builtin_ctzll(past);
            segment.sequence = base + at;
            segment.blocks = static_cast<int>(lane_value(mine, at));
            const std::int64_t sequence_start = (before + lane_value(sum, at) - segment.blocks) * heads;
            segment.item = static_cast<int>((begin - sequence_start) / segment.blocks);
            segment.start = sequence_start + static_cast<std::int64_t>(segment.item) * segment.blocks;
            segment.first = static_cast<int>(begin - segment.start);
            break;
        }
        before += lane_value(sum, kWave - 1);
    }
    segment.length = length_of(p, segment.sequence);
    segment.end = static_cast<int>(min(static_cast<std::int64_t>(segment.blocks), segment.first + length));
    return true;
}

// The segment after one that ends its sequence and head before block `end` of all; false
// where there is none.
__device__ __forceinline__ bool next_segment(const DecodeParams& p, Segment& s, std::int64_t end) {
    s.start += s.blocks;
    if (s.start >= end) return false;
    s.first = 0;
    if (++s.item == p.cache.kv_heads * p.tiles) {
        s.item = 0;
        if (++s.sequence >= p.batch) return false;
        s.length = length_of(p, s.sequence);
        s.blocks = max((s.length + kCacheKeys - 1) / kCacheKeys, 1);
    }
    s.end = static_cast<int>(min(static_cast<std::int64_t>(s.blocks), end - s.start));
    return true;
}

// 4 bytes per lane into LDS at lds_address + 4 * lane (see load_to_lds).
__device__ __forceinline__ void load_dwords_to_lds(int4v rsrc, unsigned lds_address, int voffset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(lds_address), "v"(voffset), "s"(rsrc)
                 : "memory");
}

template <int kGroups, bool kBf16>
__global__ __launch_bounds__(kThreads, kGroupsPerUnit) void cache4_attention_kernel(const DecodeParams p) {
    constexpr int kDP = 64 * kGroups;
    constexpr int kBlockBytes = cache_block_bytes(kGroups);
    constexpr int kLoads = 3 * kGroups;  // of a block: 2 kGroups KiB of codes, then 256-byte pieces of parameters
    __shared__ __attribute__((aligned(16))) unsigned char lds_blocks[kWaves][kSlots][kBlockBytes];  // a ring per wave
    __shared__ __attribute__((aligned(16))) float lds_o[kWaves][kTileRows][kCacheGroup];
    __shared__ float lds_ml[kWaves][kTileRows][2];
    __shared__ int lds_last;

    const int tid = threadIdx.x;
    const int lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15;  // token of a score block / feature quarter (A operands), query row (B operands, results)
    const int g = lane >> 4;
    Segment segment;
    std::int64_t range_length;
    const int range = blockIdx.x;
    if (!first_segment(p, range, lane, segment, range_length)) return;
    const std::int64_t range_end = (range + std::int64_t{1}) * range_length;
    const int d = p.d;
    const int per_page = p.cache.page_size / kCacheKeys;

    // -------------------------------------------------- blocks of a segment
    // A wave takes blocks first + wave, + kWaves, ... of a segment. Lane l of the window
    // holds the page of number window + l of the sequence.
    int step, page, inside, window, window_page;
    const std::int32_t* table;
    const std::uint8_t* head_data;
    auto load_window = [&]() __attribute__((always_inline)) {
        window = page;
        const int pages = (segment.length + p.cache.page_size - 1) / p.cache.page_size;
        window_page = window + lane < pages ? table[window + lane] : -1;
        // Waited for here, once in 64 pages: read in the loop as a load that may be under way,
        // it would make every block wait for all of the blocks' loads.
        wait_vmcnt<0>();
    };
    const std::uint8_t* data = nullptr;
    int bytes = 0;  // of the block at data: 0 past the segment's last, whose loads then touch no memory
    // From `step` on, the first block whose page is one of the cache.
    auto find = [&]() __attribute__((always_inline)) {
        while (step < segment.end) {
            if (page - window >= kWave) load_window();
            const int number = __builtin_amdgcn_readlane(window_page, page - window);
            if (number >= 0 && number < p.cache.pages) {
                data = head_data + number * p.cache.page_bytes + inside * kBlockBytes;
                bytes = kBlockBytes;
                return;
            }
            step += kWaves;
            inside += kWaves;
            while (inside >= per_page) inside -= per_page, ++page;
        }
        bytes = 0;
    };
    auto next_block = [&]() __attribute__((always_inline)) {
        step += kWaves;
        inside += kWaves;
        while (inside >= per_page) inside -= per_page, ++page;
        find();
    };
    // The block at data into a slot of the wave's ring; past the segment's end zeros, so
    // that the number of loads under way is always known.
    const unsigned ring = lds_address_of(&lds_blocks[wave][0][0]);
    auto issue = [&](int slot) __attribute__((always_inline)) {
        const int4v rs = make_rsrc(data, bytes);
        const unsigned to = ring + slot * kBlockBytes;
#pragma unroll
        for (int x = 0; x < 2 * kGroups; ++x) load_to_lds(rs, to + 1024 * x, 16 * lane, 1024 * x);
#pragma unroll
        for (int x = 0; x < kGroups; ++x)
            load_dwords_to_lds(rs, to + cache_key_params_at(kGroups) + 256 * x, cache_key_params_at(kGroups) + 256 * x + 4 * lane);
    };

    // ------------------------------------------------------------ a segment
    int steps[kSlots];  // of the blocks in the ring, the one to be computed first
    int slot = 0;       // its place
    uint4v qf[kGroups][2];
    int rows = 0, head0 = 0;
    // Queries and the wave's first blocks of `segment`, on their way.
    auto begin_segment = [&]() __attribute__((always_inline)) {
        const int head = segment.item / p.tiles, tile = segment.item - head * p.tiles;
        rows = min(p.group - tile * kTileRows, kTileRows);
        head0 = head * p.group + tile * kTileRows;
        table = p.table + segment.sequence * p.table_stride;
        head_data = p.cache.data + head * p.cache.head_bytes;
        step = segment.first + wave;
        page = step / per_page;
        inside = step - page * per_page;
        load_window();
#pragma unroll
        for (int m = 0; m < kGroups; ++m)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int feature = 64 * m + 16 * g + 8 * w;
                qf[m][w] = uint4v{0u, 0u, 0u, 0u};
                if (r < rows && feature < d)
                    qf[m][w] = *reinterpret_cast<const uint4v*>(p.Q + segment.sequence * p.q.row + (head0 + r) * p.q.head + feature);
            }
        find();
        slot = 0;
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the ring is read
#pragma unroll
        for (int x = 0; x < kSlots - 1; ++x) {
            if (x > 0) next_block();
            steps[x] = step;
            issue(x);
        }
    };
    const Codes<kBf16> key_codes;
    const Codes<true> value_codes;
    const uint4v ones{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    begin_segment();
    for (bool more = true; more;) {
    float q_sum[kGroups];  // of the row's features
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        q_sum[m] = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
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

    auto compute = [&](int at_step) __attribute__((always_inline)) {
        const unsigned char* const block = &lds_blocks[wave][slot][0];
        // Slot e of group g: token 16 (e / 4) + 4 g + e % 4 of the block, at place 8 g + e.
        auto params_of = [&](int which, int m, int x) __attribute__((always_inline)) {
            return *reinterpret_cast<const uint4v*>(block + cache_key_params_at(kGroups) + 128 * (which * kGroups + m) + 32 * g + 16 * x);
        };
        float4v s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            std::uint32_t words[kGroups];  // of token 16 b + r
#pragma unroll
            for (int m = 0; m < kGroups; ++m)
                words[m] = *reinterpret_cast<const std::uint32_t*>(block + cache_key_params_at(kGroups) + 128 * m +
                                                                   4 * (8 * (r >> 2) + 4 * b + (r & 3)));
            std::uint32_t k[2 * kGroups];  // codes of the lane's features of token 16 b + r
            if constexpr (kGroups == 2) {
                const uint4v codes = *reinterpret_cast<const uint4v*>(block + 64 * (16 * b + r) + 16 * g);
#pragma unroll
                for (int w = 0; w < 4; ++w) k[w] = codes[w];
            } else {
                const uint2v codes = *reinterpret_cast<const uint2v*>(block + 32 * (16 * b + r) + 8 * g);
                k[0] = codes[0], k[1] = codes[1];
            }
            const uint4v params = kGroups == 2 ? uint4v{words[0], words[kGroups - 1], words[0], words[kGroups - 1]}
                                               : uint4v{words[0], words[0], 0u, 0u};
            s[b] = mfma_16x16x32<true>(params, q_sums, float4v{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int m = 0; m < kGroups; ++m) {
                const float start = -16.0f * q_sum[m];
                float4v acc{start, start, start, start};
#pragma unroll
                for (int w = 0; w < 2; ++w) acc = mfma_16x16x32<kBf16>(key_codes.all(k[2 * m + w]), qf[m][w], acc);
                const uint4v scales = params_of(0, m, b);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[b][i] = __builtin_fmaf(half_of<true, 0>(scales[i]), acc[i], s[b][i]);
            }
        }
        // Past the length the block may hold anything, NaN included. The compiler must
        // not turn these branches into selects: one block in a sequence takes them.
        const int left = segment.length - at_step * kCacheKeys;  // tokens from the block's first on
        if (left < kCacheKeys) {
            int mine = left - 4 * g;
            asm volatile("" : "+v"(mine));
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (16 * (e / 4) + e % 4 >= mine) s[e / 4][e % 4] = -INFINITY;
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
            uint4v v_params[2] = {params_of(1, m, 0), params_of(1, m, 1)};
            if (left < kCacheKeys) {
                int mine = left - 4 * g;
                asm volatile("" : "+v"(mine));
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (16 * (e / 4) + e % 4 >= mine) v_params[e / 4][e % 4] = 0u;
            }
            uint4v high, low;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float scaled[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int e = 2 * t + x;
                    const std::uint32_t params = v_params[e / 4][e % 4];
                    scaled[x] = prob[e] * half_of<true, 0>(params);
                    below[m] = __builtin_fmaf(prob[e], half_of<true, 1>(params), below[m]);
                }
                high[t] = pack_pair<true>(scaled[0], scaled[1]);
                low[t] = pack_pair<true>(scaled[0] - half_of<true, 0>(high[t]), scaled[1] - half_of<true, 1>(high[t]));
            }
            const uint4v v = *reinterpret_cast<const uint4v*>(block + cache_values_at(kGroups) + 64 * (16 * m + r) + 16 * g);
            const uint4v a0 = value_codes.template of<0>(v), a1 = value_codes.template of<1>(v), a2 = value_codes.template of<2>(v),
                         a3 = value_codes.template of<3>(v);
            for (const uint4v& part_of_p : {high, low}) {
                o[m][0] = mfma_16x16x32<true>(a0, part_of_p, o[m][0]);
                o[m][1] = mfma_16x16x32<true>(a1, part_of_p, o[m][1]);
                o[m][2] = mfma_16x16x32<true>(a2, part_of_p, o[m][2]);
                o[m][3] = mfma_16x16x32<true>(a3, part_of_p, o[m][3]);
                sixteen[m] = mfma_16x16x32<true>(ones, part_of_p, sixteen[m]);
            }
        }
    };
    // Every wave leaves when its blocks run out.
    while (steps[0] < segment.end) {
        next_block();
        steps[kSlots - 1] = step;
        // The slot that the block before was read from: those reads are done.
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        issue(slot == 0 ? kSlots - 1 : slot - 1);
        wait_vmcnt<(kSlots - 1) * kLoads>();  // all but the kSlots - 1 blocks after this one
        asm volatile("" ::: "memory");
        compute(steps[0]);
#pragma unroll
        for (int x = 0; x + 1 < kSlots; ++x) steps[x] = steps[x + 1];
        slot = slot + 1 == kSlots ? 0 : slot + 1;
    }
    const Segment done = segment;
    const int done_rows = rows, done_head0 = head0;
    more = segment.end == segment.blocks && next_segment(p, segment, range_end);
    if (more) begin_segment();

    // ------------------------------------------------------- merge of waves
    row_sum = groups_sum(row_sum);
    if (g == 0) {
        lds_ml[wave][r][0] = row_max;
        lds_ml[wave][r][1] = row_sum;
    }
    const int row = tid >> 4, f0 = 4 * (tid & 15);  // of every group
    float row_m = -INFINITY, row_l = 0.0f;
    float weight[kWaves];
    float4v acc[kGroups];
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        const float rest = __builtin_fmaf(-16.0f, sixteen[m][0], groups_sum(below[m]));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4v*>(&lds_o[wave][r][16 * g + 4 * i]) =
                float4v{o[m][0][i] + rest, o[m][1][i] + rest, o[m][2][i] + rest, o[m][3][i] + rest};
        __syncthreads();
        if (m == 0) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) row_m = fmaxf(row_m, lds_ml[w][row][0]);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                // (A wave whose scores are all NaN has the maximum -inf, and a NaN sum.)
                const float m_w = lds_ml[w][row][0];
                weight[w] = m_w == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_w - row_m);
                row_l += weight[w] * lds_ml[w][row][1];
            }
        }
        acc[m] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) acc[m] += weight[w] * *reinterpret_cast<const float4v*>(&lds_o[w][row][f0]);
        __syncthreads();  // lds_o is read: the next group or segment may write it
    }
    const bool mine = row < done_rows;

    // ------------------------------------------------------- merge of parts
    // The ranges that have a part of this sequence and head: part i is the continued one
    // of range first_range + i, part 0 the one to be continued.
    bool whole = true;
    const int first_range = static_cast<int>(done.start / range_length);
    const int count = static_cast<int>((done.start + done.blocks - 1) / range_length) - first_range + 1;
    if (count > 1) {
        constexpr int kPartO = kTileRows * kDP, kPartMl = kTileRows * 2;
        const Rsrc ro = shared_rows(p.part_o, std::int64_t{2} * kRanges * kPartO);
        const Rsrc rml = shared_rows(p.part_ml, std::int64_t{2} * kRanges * kPartMl);
        auto place_of = [&](int i) { return 2 * (first_range + i) + (i == 0 ? 1 : 0); };
        if (mine) {
            const int at = place_of(range - first_range);
#pragma unroll
            for (int x = 0; x < kGroups; ++x)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4v, acc[x]), ro,
                                                       (at * kPartO + row * kDP + 64 * x + f0) * 4, 0, kDeviceScope);
            if (f0 == 0)
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uint2v, float2v{row_m, row_l}), rml,
                                                      (at * kPartMl + 2 * row) * 4, 0, kDeviceScope);
        }
        whole = last_arrival(p.arrivals + first_range, count, &lds_last);
        if (whole && mine) {
            row_m = -INFINITY;
            row_l = 0.0f;
#pragma unroll
            for (int x = 0; x < kGroups; ++x) acc[x] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            constexpr int kBatch = 8;
            for (int s0 = 0; s0 < count; s0 += kBatch) {
                float2v state[kBatch];
                float4v value[kBatch][kGroups];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int at = place_of(min(s0 + u, count - 1));
                    state[u] = __builtin_bit_cast(
                        float2v, __builtin_amdgcn_raw_buffer_load_b64(rml, (at * kPartMl + 2 * row) * 4, 0, kDeviceScope));
#pragma unroll
                    for (int x = 0; x < kGroups; ++x)
                        value[u][x] = __builtin_bit_cast(
                            float4v, __builtin_amdgcn_raw_buffer_load_b128(ro, (at * kPartO + row * kDP + 64 * x + f0) * 4, 0,
                                                                           kDeviceScope));
                }
                merge_batch<kBatch, true>(
                    row_m, row_l, count - s0, [&](int u) __attribute__((always_inline)) { return state[u]; },
                    [&](int u, PartWeights w) __attribute__((always_inline)) {
#pragma unroll
                        for (int x = 0; x < kGroups; ++x) acc[x] = merged(acc[x], value[u][x], w);
                    });
            }
        }
    }
    if (whole && mine) {
        const float inverse = row_l == 0.0f ? 0.0f : 1.0f / row_l;  // 0: no token
        std::uint16_t* const out = p.O + done.sequence * p.o.row + (done_head0 + row) * p.o.head + f0;
#pragma unroll
        for (int x = 0; x < kGroups; ++x)
            if (64 * x + f0 < d)
                *reinterpret_cast<uint2v*>(out + 64 * x) = uint2v{pack_pair<kBf16>(acc[x][0] * inverse, acc[x][1] * inverse),
                                                                 pack_pair<kBf16>(acc[x][2] * inverse, acc[x][3] * inverse)};
    }
    }
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
    p.part_o = reinterpret_cast<float*>(p.arrivals + kRanges);
    p.part_ml = p.part_o + std::size_t{2} * kRanges * kTileRows * kCacheGroup * p.cache.groups;
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
    // Ranges of at least kLeastSteps blocks.
    const std::int64_t items = static_cast<std::int64_t>(a.batch) * a.kv_heads * p.tiles;
    const std::int64_t most = (p.most_tokens - 1) / kCacheKeys + 1;  // blocks of one of them
    p.ranges = static_cast<int>(std::min<std::int64_t>(kRanges, items > kRanges * kLeastSteps ? kRanges : (items * most - 1) / kLeastSteps + 1));
    const hipError_t found = check_device();
    if (found != hipSuccess) return found;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool bf16 = a.dtype == TILEMIX_DTYPE_BF16;
    const unsigned workgroups = static_cast<unsigned>(p.ranges);
    if (p.cache.groups == 1)
        bf16 ? cache4_attention_kernel<1, true><<<workgroups, kThreads, 0, s>>>(p)
             : cache4_attention_kernel<1, false><<<workgroups, kThreads, 0, s>>>(p);
    else
        bf16 ? cache4_attention_kernel<2, true><<<workgroups, kThreads, 0, s>>>(p)
             : cache4_attention_kernel<2, false><<<workgroups, kThreads, 0, s>>>(p);
    return hipGetLastError();
}
