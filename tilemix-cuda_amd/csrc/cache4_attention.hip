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
// fp32 sums; of p scale, two bf16 parts (hi + lo, 2^-16 of it) are multiplied, as
// bf16 holds any scale (fp16 would not).
//
// What bounds it is memory: 144 bytes a token and head at d = 128. The cache lies
// in blocks of 32 tokens in the order of these operands (serving.h): a wave takes
// a block per step, from a ring of LDS slots of its own that LDS DMA fills in
// contiguous KiB pieces while the block before is computed. (Held in registers, a block ahead
// does not fit beside the accumulators without spills.)
//
// Split of the work: the blocks of all sequences and heads, one after the other, are
// cut into ranges of equal length, one per workgroup (two or three a CU, one round),
// found on the device from the lengths (first_segment): lengths differ, and the host does not
// know them. A range is a series of segments - blocks of one sequence and head; a
// segment's queries and first blocks are on their way while the one before is merged over
// the waves. Only a range's first and last segment can be a part of a sequence and
// head: those go to the workspace, where the workgroup that arrives last merges them in order.
//
// Measured: 64 sequences of 1 to 16384 tokens, 32 query and 8 key heads x 128: 93 us, 4.5 TB/s;
// 2 of 32768 tokens, 16 heads: 35 to 39 us, 3.9 to 4.3 TB/s; 64 of 8192 tokens, 8 key heads, 5.2 TB/s. A
// range's start and end take about 6 us. One sequence of 1003
// tokens, 4 key heads x 64: 9.7 us.

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
// Workgroups of a CU: three of 8 rows (their LDS is just under a third), two of 16. (128
// sequences of up to 200 tokens, 8 key heads x 128: two 23 us, three 20; of up to 2048 41 and 38; two of
// 32768, 16 heads, 35.7 and 36.4.)
constexpr int groups_per_unit(int rows) { return rows == 8 ? 3 : 2; }
constexpr int kSlots = 2;       // blocks in a wave's ring, the one computed and the next (three: 0 to 6 % more time)
constexpr int kTileRows = 16;   // query rows of a workgroup
constexpr int kLeastSteps = 8;  // places of a range at least
constexpr int kSwitch = 8;      // places of a range that the step to another sequence counts for
constexpr int kRanges = 768;    // at most: workgroups that the device holds at once
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

// Sum over the four lanes r, r + 16, r + 32, r + 48, in each of them.
__device__ __forceinline__ void permlane16_swap(float& a, float& b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ float groups_sum(float x) {
    float a = x, b = x;
    permlane16_swap(a, b);
    a = a + b;
    b = a;
    permlane32_swap(a, b);
    return a + b;
}

// f over the 16 lanes of a row, in each of them (DPP: quad partners, then mirrored).
template <typename F>
__device__ __forceinline__ float over_16_lanes(float x, F&& f) {
    auto step = [&](auto control) __attribute__((always_inline)) {
        constexpr int kControl = decltype(control)::value;
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kControl, 0xf, 0xf, false));
    };
    x = f(x, step(std::integral_constant<int, 0xb1>{}));
    x = f(x, step(std::integral_constant<int, 0x4e>{}));
    x = f(x, step(std::integral_constant<int, 0x141>{}));
    return f(x, step(std::integral_constant<int, 0x140>{}));
}

__device__ __forceinline__ unsigned lane_value(unsigned v, int lane) {
    return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

__device__ __forceinline__ int length_of(const DecodeParams& p, int b) { return min(max(p.lengths[b], 0), p.most_tokens); }
// Blocks of sequence b. An empty one counts as one block (without a page), so that some
// range has it and writes its zeros.
__device__ __forceinline__ int blocks_of(int length) { return max((length + kCacheKeys - 1) / kCacheKeys, 1); }

// Positions: the sequences of head 0, then of head 1, ... (a head: one key head's row
// tile), each with its blocks and `gap` places more, which stand for the time that a
// workgroup takes from one sequence to the next. With a sequence's heads side by side, a
// short one's would all fall to the same workgroup (64 sequences of 1 to 16384 tokens, 8
// heads: 121 us so, 93 as it is). All positions fit 30 bits (checked by the host).
struct Segment {
    int sequence, head;
    int first, end, blocks;  // blocks first .. end - 1 of the sequence's
    int length;              // tokens of the sequence
    int start;               // position of its first block
};

struct Plan {
    int length;  // of a range
    int gap;
};

// The ranges, and the segment in which range number `range` begins; false where it has
// none. Wave-uniform.
__device__ __forceinline__ bool first_segment(const DecodeParams& p, int range, int lane, Segment& segment, Plan& plan) {
    const unsigned heads = p.cache.kv_heads * p.tiles;
    auto blocks_at = [&](int b) __attribute__((always_inline)) { return b < p.batch ? blocks_of(length_of(p, b)) : 0; };
    const int kept = blocks_at(lane);  // of the first kWave sequences
    const int sequence0 = __builtin_amdgcn_readfirstlane(kept);
    bool alike = __all(kept == sequence0 || lane >= p.batch);
    unsigned blocks = lane_value(prefix_sum(kept), kWave - 1);  // of a head
    for (int base = kWave; base < p.batch; base += kWave) {
        const int mine = blocks_at(base + lane);
        alike = alike && __all(mine == sequence0 || base + lane >= p.batch);
        blocks += lane_value(prefix_sum(mine), kWave - 1);
    }
    plan.gap = kSwitch;
    unsigned one = blocks + p.batch * kSwitch, total = one * heads;
    // A range of n places takes about as long as the merge of n parts does (of one key head's
    // 1024 blocks, ranges of 8 places: 22.7 us, 22 19.0, 32 19.7; of 128, 8 places 12.0, 16 13.0).
    const int least = max(static_cast<int>(sqrtf(0.5f * static_cast<float>(one) / static_cast<float>(p.batch))), kLeastSteps);
    plan.length = max(static_cast<int>((total + p.ranges - 1) / p.ranges), least);
    const unsigned items = p.batch * heads, ranges = p.ranges;
    // Sequences that are all alike: whole ranges for each sequence and head, or whole sequences for
    // a range, so that no range ends inside one, if that is hardly more for each or leaves at
    // least two of three workgroups (2 sequences of 32768 tokens, 16 heads: 40.7 us cut anywhere,
    // 35.4 so; 64 of 2048, 8 heads: 37.8 and 33.2; 128, 8 heads, of 1024: 43.0 and 37.7). One a
    // few blocks shorter than the others, or empty, has them cut anywhere: 32768 and 32700 tokens
    // 37.7 us for 34.6, 128 of 985 to 1024 42.1 for 35.8.
    if (alike && items <= ranges) {
        const unsigned each = ranges / items;
        const int length = max(static_cast<int>((sequence0 + each - 1) / each), least);
        if (length <= plan.length + kSwitch || 3 * items * each >= 2 * ranges) {
            plan.gap = (length - sequence0 % length) % length;
            plan.length = length;
            one = blocks + p.batch * plan.gap;
            total = one * heads;
        }
    } else if (alike) {
        const unsigned each = (items - 1) / ranges + 1;
        if (3 * ((items - 1) / each + 1) >= 2 * ranges) plan.length = each * (sequence0 + kSwitch);
    }
    const unsigned begin = static_cast<unsigned>(range) * plan.length;
    if (begin >= total) return false;
    segment.head = static_cast<int>(begin / one);
    const unsigned inside = begin - segment.head * one;
    unsigned before = 0;
    for (int base = 0;; base += kWave) {
        const unsigned mine = base == 0 ? kept : blocks_at(base + lane);
        const unsigned sum = prefix_sum(base + lane < p.batch ? mine + plan.gap : 0u) + before;
        const std::uint64_t past = __ballot(sum > inside);
        if (past) {
            const int at = __builtin_ctzll(past);
            segment.sequence = base + at;
            segment.blocks = static_cast<int>(lane_value(mine, at));
            segment.start = static_cast<int>(segment.head * one + lane_value(sum, at)) - segment.blocks - plan.gap;
            segment.first = static_cast<int>(begin) - segment.start;
            break;
        }
        before = lane_value(sum, kWave - 1);
    }
    segment.end = min(segment.blocks, segment.first + plan.length);
    return true;
}

// 4 bytes per lane into LDS at lds_address + 4 * lane (see load_to_lds).
__device__ __forceinline__ void load_dwords_to_lds(int4v rsrc, unsigned lds_address, int voffset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(lds_address), "v"(voffset), "s"(rsrc)
                 : "memory");
}

// kRows: query rows of a workgroup, 8 or 16. Scores are taken with queries as the rows
// and tokens as the columns of a tile, so that a lane has 4 rows of a token (of two with
// 16 rows), and its scale and minimum once; with 8 rows the two halves of a
// tile are the same rows, and hold the two 16-token halves of a block.
template <int kGroups, bool kBf16, int kRows>
__global__ __launch_bounds__(kThreads, groups_per_unit(kRows)) void cache4_attention_kernel(const DecodeParams p) {
    constexpr int kTiles = kRows / 8;  // tokens of a lane
    constexpr int kDP = 64 * kGroups;
    constexpr int kBlockBytes = cache_block_bytes(kGroups);
    constexpr int kLoads = 3 * kGroups;  // of a block: 2 kGroups KiB of codes, then 256-byte pieces of parameters
    __shared__ __attribute__((aligned(16))) unsigned char lds_blocks[kWaves][kSlots][kBlockBytes];  // a ring per wave
    // A wave's piece: p scale on its way to the matrix operand's layout while blocks are computed,
    // O at a segment's end.
    constexpr int kPieceBytes = kRows * kDP * 4;
    static_assert(kPieceBytes >= kGroups * 2 * kRows * kCacheKeys * 2, "p scale fits");
    __shared__ __attribute__((aligned(16))) unsigned char lds_piece[kWaves][kPieceBytes];
    __shared__ __attribute__((aligned(16))) float lds_ml[kWaves][kRows][4];  // maximum, sum, sum p minimum of both groups
    int* const lds_last = reinterpret_cast<int*>(&lds_ml[0][0][0]);  // [2], at the end

    const int tid = threadIdx.x;
    const int lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15;  // token of a score block / feature quarter (A operands), query row (B operands, results)
    const int g = lane >> 4;
    // The lane's rows row0 .. + 3, its (first) token of a block and that token's place.
    const int row0 = 4 * g % kRows, token0 = r + (kTiles == 1 ? 16 * (g >> 1) : 0), place0 = cache_place(token0);
    // Over the lanes that hold the same rows.
    auto row_reduce = [&](float x, auto&& f) __attribute__((always_inline)) {
        x = over_16_lanes(x, f);
        if constexpr (kTiles == 1) {
            float y = x;
            permlane32_swap(x, y);
            x = f(x, y);
        }
        return x;
    };
    Segment segment;
    Plan plan;
    const int range = blockIdx.x;
    if (!first_segment(p, range, lane, segment, plan)) return;
    const int range_end = (range + 1) * plan.length;
    const int d = p.d;
    const int per_page = p.cache.page_size / kCacheKeys;

    // Lengths of sequences lengths_at .. + 63, one a lane.
    int lengths_at = segment.sequence;
    int lengths = lengths_at + lane < p.batch ? length_of(p, lengths_at + lane) : 0;
    segment.length = __builtin_amdgcn_readfirstlane(lengths);
    // The segment after `s` in this range.
    auto after = [&](const Segment& s, Segment& out) __attribute__((always_inline)) {
        out = s;
        out.start += s.blocks + plan.gap;
        if (s.end < s.blocks || out.start >= range_end) return false;
        out.first = 0;
        if (++out.sequence == p.batch) {
            out.sequence = 0;
            if (++out.head == p.cache.kv_heads * p.tiles) return false;
        }
        if (static_cast<unsigned>(out.sequence - lengths_at) >= kWave) {
            lengths_at = out.sequence;
            lengths = lengths_at + lane < p.batch ? length_of(p, lengths_at + lane) : 0;
        }
        out.length = __builtin_amdgcn_readlane(lengths, out.sequence - lengths_at);
        out.blocks = blocks_of(out.length);
        out.end = min(out.blocks, range_end - out.start);
        return true;
    };
    // A range that begins in the places after a sequence's blocks begins with the next one.
    if (segment.first >= segment.blocks) {
        segment.end = segment.blocks;
        const Segment before = segment;
        if (!after(before, segment)) return;
    }
    auto head_of = [&](const Segment& s) __attribute__((always_inline)) { return p.tiles == 1 ? s.head : s.head / p.tiles; };

    // ------------------------------------------------- a wave's blocks, in turn
    // Blocks first + wave, + kWaves, ... of a segment, then of the next: a segment's first
    // blocks are under way before the one before is done. Lane l of the window holds
    // page number window + l of the sequence.
    int step, end, page, inside, pages, window, window_page;
    const std::int32_t* table;
    const std::uint8_t* head_data;
    const std::uint8_t* data = nullptr;
    int bytes = 0;  // of the block at data; 0: none, and its loads touch no memory
    auto load_window = [&]() __attribute__((always_inline)) {
        window = page;
        window_page = window + lane < pages ? table[window + lane] : -1;
        // Waited for here, once in 64 pages: read in the loop as a load that may be under way,
        // it would make every block wait for all of the blocks' loads.
        wait_vmcnt<0>();
    };
    auto pages_of = [&](const Segment& s) __attribute__((always_inline)) {
        return s.length == 0 ? 0 : static_cast<int>(static_cast<unsigned>(s.length - 1) / static_cast<unsigned>(p.cache.page_size)) + 1;
    };
    auto enter = [&](const Segment& s) __attribute__((always_inline)) {
        table = p.table + s.sequence * p.table_stride;
        head_data = p.cache.data + head_of(s) * p.cache.head_bytes;
        pages = pages_of(s);
        end = s.end;
        step = s.first + wave;
        page = step / per_page;
        inside = step - page * per_page;
    };
    // From `step` on, the first block whose page is one of the cache.
    auto find = [&]() __attribute__((always_inline)) {
        bytes = 0;
        while (step < end) {
            if (page - window >= kWave) load_window();
            const int number = __builtin_amdgcn_readlane(window_page, page - window);
            if (number >= 0 && number < p.cache.pages) {
                data = head_data + cache_block_at(number, p.cache.page_bytes, inside, kBlockBytes);
                bytes = kBlockBytes;
                return;
            }
            step += kWaves;
            inside += kWaves;
            while (inside >= per_page) inside -= per_page, ++page;
        }
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

    // Queries of a segment: row r (mod kRows) of its tile.
    auto load_queries = [&](uint4v (&to)[kGroups][2], const Segment& s) __attribute__((always_inline)) {
        const int head = head_of(s), tile = s.head - head * p.tiles;
        const int query = tile * kTileRows + r % kRows;
        const std::uint16_t* const from = p.Q + s.sequence * p.q.row + (head * p.group + query) * p.q.head;
#pragma unroll
        for (int m = 0; m < kGroups; ++m)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int feature = 64 * m + 16 * g + 8 * w;
                to[m][w] = query < p.group && feature < d ? *reinterpret_cast<const uint4v*>(from + feature) : uint4v{0u, 0u, 0u, 0u};
            }
    };
    // What follows `segment`: its queries and the window of the wave's first pages are loaded
    // while `segment` is computed.
    Segment next;
    bool has_next, in_next = false;  // in_next: the wave's blocks have got to `next`
    int next_page = 0;
    uint4v qf[kGroups][2], next_qf[kGroups][2];
    auto look_ahead = [&]() __attribute__((always_inline)) {
        has_next = after(segment, next);
        if (has_next) {
            const int count = pages_of(next), first = wave / per_page;
            next_page = first + lane < count ? p.table[next.sequence * p.table_stride + first + lane] : -1;
            load_queries(next_qf, next);
        }
    };
    // The ring: what each slot holds, the one to be computed first. Steps of `segment`,
    // kInNext more for those of `next`, kNone.
    constexpr int kInNext = 1 << 28, kNone = -1;
    int held[kSlots];
    int slot = 0;  // place of held[0]
    auto take_next = [&](int to) __attribute__((always_inline)) {
        if (bytes == 0 && !in_next && has_next) {
            enter(next);
            window = page;
            window_page = next_page;
            in_next = true;
            find();
        }
        issue(to);
        const int what = bytes == 0 ? kNone : step + (in_next ? kInNext : 0);
        if (bytes != 0) {
            step += kWaves;
            inside += kWaves;
            while (inside >= per_page) inside -= per_page, ++page;
            find();
        }
        return what;
    };
    const Codes<kBf16> key_codes;
    const Codes<true> value_codes;
    const uint4v ones{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    // What the range has a part of, at most two: merged, where this workgroup is the last
    // to arrive, at the end.
    struct Shared {
        Segment segment;
        std::uint16_t* out;
    };
    Shared shared[2];
    int shares = 0;
    // A thread's row and 4 kPasses features in the merges
    // (with 8 rows of 64 features half of the threads have none).
    constexpr int kThreadsPerRow = kThreads / kRows < kDP / 4 ? kThreads / kRows : kDP / 4, kPasses = kDP / 4 / kThreadsPerRow;
    const bool has_row = tid / kThreadsPerRow < kRows;
    const int row = has_row ? tid / kThreadsPerRow : 0, f0 = 4 * (tid % kThreadsPerRow);
    auto feature_of = [&](int pass) __attribute__((always_inline)) { return f0 + 4 * kThreadsPerRow * pass; };
    auto rows_of = [&](const Segment& s) __attribute__((always_inline)) {
        return min(p.group - (s.head - head_of(s) * p.tiles) * kTileRows, kRows);
    };
    auto store_rows = [&](const float4v (&value)[kPasses], float l, std::uint16_t* out) __attribute__((always_inline)) {
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;  // 0: no token
#pragma unroll
        for (int x = 0; x < kPasses; ++x)
            if (feature_of(x) < d)
                *reinterpret_cast<uint2v*>(out + row * p.o.head + feature_of(x)) =
                    uint2v{pack_pair<kBf16>(value[x][0] * inverse, value[x][1] * inverse),
                           pack_pair<kBf16>(value[x][2] * inverse, value[x][3] * inverse)};
    };
    // Parts in the workspace: part i of a sequence and head is the continued one of range
    // first_range + i, part 0 the one to be continued.
    constexpr int kPartO = kTileRows * kDP, kPartMl = kTileRows * 2;
    const Rsrc ro = shared_rows(p.part_o, std::int64_t{2} * kRanges * kPartO);
    const Rsrc rml = shared_rows(p.part_ml, std::int64_t{2} * kRanges * kPartMl);
    auto part_place = [](int first_range, int i) { return 2 * (first_range + i) + (i == 0 ? 1 : 0); };
    auto part_at = [&](int place, int pass) __attribute__((always_inline)) { return (place * kPartO + row * kDP + feature_of(pass)) * 4; };

    enter(segment);
    load_window();
    load_queries(qf, segment);
    look_ahead();
    find();
#pragma unroll
    for (int x = 0; x < kSlots - 1; ++x) held[x] = take_next(x);
    for (;;) {
    // q_sum[m][i]: of the features of row row0 + i.
    float4v q_sum[kGroups];
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        float sum = 0.0f;  // of row r
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (p.negate) qf[m][w] ^= 0x80008000u;
#pragma unroll
            for (int x = 0; x < 4; ++x) sum += half_of<kBf16, 0>(qf[m][w][x]) + half_of<kBf16, 1>(qf[m][w][x]);
        }
        sum = groups_sum(sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) q_sum[m][i] = __shfl(sum, row0 + i);
    }

    float4v o[kGroups][4];     // o[m][f][i]: column r, feature 64 m + 16 g + 4 i + f
    float4v sixteen[kGroups];  // sum p scale, as multiplied, of column r in every element
    float4v below[kGroups];    // of the lane's tokens: sum p minimum,
    float4v row_sum{0.0f, 0.0f, 0.0f, 0.0f};  // and sum p,
    float4v row_max{-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // of the rows row0 + i
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        below[m] = sixteen[m] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int f = 0; f < 4; ++f) o[m][f] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto compute = [&](int at_step) __attribute__((always_inline)) {
        const unsigned char* const block = &lds_blocks[wave][slot][0];
        const int left = segment.length - at_step * kCacheKeys;  // tokens from the block's first on
        float4v s[kTiles];       // rows row0 + i of the tile's token of the lane
        std::uint32_t v_params[kTiles][kGroups];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) s[t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        std::uint32_t k[2][2 * kGroups];  // codes of the lane's features of token 16 b + r
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if constexpr (kGroups == 2) {
                const uint4v codes = *reinterpret_cast<const uint4v*>(block + 64 * (16 * b + r) + 16 * g);
#pragma unroll
                for (int w = 0; w < 4; ++w) k[b][w] = codes[w];
            } else {
                const uint2v codes = *reinterpret_cast<const uint2v*>(block + 32 * (16 * b + r) + 8 * g);
                k[b][0] = codes[0], k[b][1] = codes[1];
            }
        }
#pragma unroll
        for (int m = 0; m < kGroups; ++m) {
            float4v acc[2];  // sum (16 + code) q of rows 4 g + i (mod kRows) and token 16 b + r
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                acc[b] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < 2; ++w) acc[b] = mfma_16x16x32<kBf16>(qf[m][w], key_codes.all(k[b][2 * m + w]), acc[b]);
            }
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const unsigned char* const params = block + 4 * place0 + 16 * t + 128 * m;
                const std::uint32_t word = *reinterpret_cast<const std::uint32_t*>(params + cache_key_params_at(kGroups));
                v_params[t][m] = *reinterpret_cast<const std::uint32_t*>(params + cache_value_params_at(kGroups));
                const float scale = half_of<true, 0>(word), low = __builtin_fmaf(-16.0f, scale, half_of<true, 1>(word));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // With 8 rows the tile holds them twice: the lanes of the upper half take token 16 + r.
                    const float sum = kTiles == 2 ? acc[t][i] : g >= 2 ? acc[1][i] : acc[0][i];
                    s[t][i] = __builtin_fmaf(scale, sum, __builtin_fmaf(low, q_sum[m][i], s[t][i]));
                }
            }
        }
        // Past the length the block may hold anything, NaN included.
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
            if (token0 + 16 * t >= left) {
                s[t] = float4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int m = 0; m < kGroups; ++m) v_params[t][m] = 0u;
            }
        const float c = p.score_log2;  // > 0
        float over = -INFINITY;  // how far a score is above its row's maximum
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] *= c;
                over = fmaxf(over, s[t][i] - row_max[i]);
            }
        // (-inf - -inf is NaN, which fmaxf passes over: such a row stays as it is.)
        if (__any(over > kLazyRescale)) {
            float4v alpha;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float top = row_reduce(kTiles == 2 ? fmaxf(s[0][i], s[kTiles - 1][i]) : s[0][i], [](float x, float y) { return fmaxf(x, y); });
                const float m_new = fmaxf(row_max[i], top);
                alpha[i] = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(row_max[i] - m_new);
                row_max[i] = m_new;
            }
            row_sum *= alpha;
            // The columns' factors, through LDS.
            float* const factors = &lds_ml[wave][0][0];
            if (r == 0 && (kTiles == 2 || g < 2)) *reinterpret_cast<float4v*>(factors + row0) = alpha;
            asm volatile("" ::: "memory");
            const float factor = factors[r % kRows];
            asm volatile("" ::: "memory");
#pragma unroll
            for (int m = 0; m < kGroups; ++m) {
                below[m] *= alpha;
                sixteen[m] *= factor;
#pragma unroll
                for (int f = 0; f < 4; ++f) o[m][f] *= factor;
            }
        }
        float4v prob[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                prob[t][i] = __builtin_amdgcn_exp2f(s[t][i] - (row_max[i] == -INFINITY ? 0.0f : row_max[i]));
                row_sum[i] += prob[t][i];
            }
        // p scale in two bf16 parts, from tokens in lanes and rows in registers to the
        // matrix operand's columns: [m][part][row][place] in the wave's piece.
        std::uint16_t* const turn = reinterpret_cast<std::uint16_t*>(lds_piece[wave]);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int m = 0; m < kGroups; ++m)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const float scale = half_of<true, 0>(v_params[t][m]), low = half_of<true, 1>(v_params[t][m]);
                std::uint16_t* const to = turn + (2 * m * kRows + row0) * kCacheKeys + place0 + 4 * t;
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float x = prob[t][i] * scale, y = prob[t][i + 1] * scale;
                    const std::uint32_t first = pack_pair<true>(x, y);
                    const std::uint32_t second = pack_pair<true>(x - half_of<true, 0>(first), y - half_of<true, 1>(first));
                    to[i * kCacheKeys] = static_cast<std::uint16_t>(first);
                    to[(i + 1) * kCacheKeys] = static_cast<std::uint16_t>(first >> 16);
                    to[(kRows + i) * kCacheKeys] = static_cast<std::uint16_t>(second);
                    to[(kRows + i + 1) * kCacheKeys] = static_cast<std::uint16_t>(second >> 16);
                    below[m][i] = __builtin_fmaf(prob[t][i], low, below[m][i]);
                    below[m][i + 1] = __builtin_fmaf(prob[t][i + 1], low, below[m][i + 1]);
                }
            }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int m = 0; m < kGroups; ++m) {
            const uint4v v = *reinterpret_cast<const uint4v*>(block + cache_values_at(kGroups) + 64 * (16 * m + r) + 16 * g);
            const uint4v a0 = value_codes.template of<0>(v), a1 = value_codes.template of<1>(v), a2 = value_codes.template of<2>(v),
                         a3 = value_codes.template of<3>(v);
            // Columns: 8 rows' first parts and their second parts, or 16 rows and one part after the other.
#pragma unroll
            for (int part = 0; part < kTiles; ++part) {
                const uint4v ps = *reinterpret_cast<const uint4v*>(turn + (2 * m * kRows + part * kRows + r) * kCacheKeys + 8 * g);
                o[m][0] = mfma_16x16x32<true>(a0, ps, o[m][0]);
                o[m][1] = mfma_16x16x32<true>(a1, ps, o[m][1]);
                o[m][2] = mfma_16x16x32<true>(a2, ps, o[m][2]);
                o[m][3] = mfma_16x16x32<true>(a3, ps, o[m][3]);
                sixteen[m] = mfma_16x16x32<true>(ones, ps, sixteen[m]);
            }
        }
        asm volatile("" ::: "memory");
    };
    // Until the wave's blocks of the segment run out. (One that had none left for the ring
    // passes a place by as soon as there is a next segment to fill it from.)
    for (;;) {
        const int now = held[0];
        const bool mine = now >= 0 && now < kInNext;
        if (!mine && !(now == kNone && has_next && !in_next)) break;
        // Into the slot that the block before was read from: those reads are done.
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        held[kSlots - 1] = take_next(slot == 0 ? kSlots - 1 : slot - 1);
        if (mine) {
            wait_vmcnt<(kSlots - 1) * kLoads>();  // all but the kSlots - 1 blocks after this one
            asm volatile("" ::: "memory");
            compute(now);
        }
#pragma unroll
        for (int x = 0; x + 1 < kSlots; ++x) held[x] = held[x + 1];
        slot = slot + 1 == kSlots ? 0 : slot + 1;
    }

    // ------------------------------------------------------- merge of waves
    auto add = [](float x, float y) { return x + y; };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4v state{row_max[i], row_reduce(row_sum[i], add), 0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < kGroups; ++m) state[2 + m] = row_reduce(below[m][i], add);
        if (r == 0 && (kTiles == 2 || g < 2)) *reinterpret_cast<float4v*>(&lds_ml[wave][row0 + i][0]) = state;
    }
#pragma unroll
    for (int m = 0; m < kGroups; ++m) {
        const float rest = -16.0f * sixteen[m][0];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4v quad{o[m][0][i] + rest, o[m][1][i] + rest, o[m][2][i] + rest, o[m][3][i] + rest};
            if constexpr (kTiles == 1) {  // the second parts of p scale, 8 columns on
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                    const float x = quad[f];
                    quad[f] = x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false));
                }
            }
            if (r < kRows) *reinterpret_cast<float4v*>(lds_piece[wave] + (r * kDP + 64 * m + 16 * g + 4 * i) * 4) = quad;
        }
    }
    __syncthreads();
    float row_m = -INFINITY, row_l = 0.0f;
    float4v value[kPasses];
#pragma unroll
    for (int x = 0; x < kPasses; ++x) value[x] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) row_m = fmaxf(row_m, lds_ml[w][row][0]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        // (A wave whose scores are all NaN has the maximum -inf, and a NaN sum.)
        const float m_w = lds_ml[w][row][0];
        const float weight = m_w == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_w - row_m);
        row_l += weight * lds_ml[w][row][1];
#pragma unroll
        for (int x = 0; x < kPasses; ++x)
            value[x] += weight * (*reinterpret_cast<const float4v*>(lds_piece[w] + (row * kDP + feature_of(x)) * 4) +
                                  lds_ml[w][row][2 + feature_of(x) / kCacheGroup]);
    }
    const bool live = has_row && row < rows_of(segment);
    std::uint16_t* out;
    {
        const int head = head_of(segment), tile = segment.head - head * p.tiles;
        out = p.O + segment.sequence * p.o.row + (head * p.group + tile * kTileRows) * p.o.head;
    }
    if (segment.first == 0 && segment.end == segment.blocks) {
        if (live) store_rows(value, row_l, out);
    } else {
        const int place = 2 * range + (segment.first == 0 ? 1 : 0);
        if (live) {
#pragma unroll
            for (int x = 0; x < kPasses; ++x)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4v, value[x]), ro, part_at(place, x), 0, kDeviceScope);
            if (f0 == 0)
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uint2v, float2v{row_m, row_l}), rml,
                                                      (place * kPartMl + 2 * row) * 4, 0, kDeviceScope);
        }
        if (shares == 0)
            shared[0] = Shared{segment, out};
        else
            shared[1] = Shared{segment, out};
        ++shares;
    }
    if (!has_next) break;
    __syncthreads();  // the pieces are read: the next segment writes them
    segment = next;
    in_next = false;
#pragma unroll
    for (int x = 0; x < kSlots - 1; ++x)
        if (held[x] != kNone) held[x] -= kInNext;
#pragma unroll
    for (int m = 0; m < kGroups; ++m)
#pragma unroll
        for (int w = 0; w < 2; ++w) qf[m][w] = next_qf[m][w];
    look_ahead();
    }

    // ------------------------------------------------------- merge of parts
    if (shares == 0) return;
    // As last_arrival (attention_common.h), for both parts at once.
    auto first_range_of = [&](const Segment& s) __attribute__((always_inline)) {
        return s.first == 0 ? range : s.start / plan.length;
    };
    auto count_of = [&](const Segment& s) __attribute__((always_inline)) {
        return (s.start + s.blocks - 1) / plan.length - first_range_of(s) + 1;
    };
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (lane == 0 && wave < shares) {
        const Segment mine = wave == 0 ? shared[0].segment : shared[1].segment;
        unsigned* const counter = p.arrivals + first_range_of(mine);
        const unsigned before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = before == static_cast<unsigned>(count_of(mine)) - 1u;
        if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        lds_last[wave] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int which = 0; which < shares; ++which) {
        const Shared mine = which == 0 ? shared[0] : shared[1];
        if (!lds_last[which] || !has_row || row >= rows_of(mine.segment)) continue;
        const int first_range = first_range_of(mine.segment), count = count_of(mine.segment);
        float m_all = -INFINITY, l_all = 0.0f;
        float4v sum[kPasses];
#pragma unroll
        for (int x = 0; x < kPasses; ++x) sum[x] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int kBatch = 16 / kPasses;
        for (int s0 = 0; s0 < count; s0 += kBatch) {
            float2v state[kBatch];
            float4v part[kBatch][kPasses];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int place = part_place(first_range, min(s0 + u, count - 1));
                state[u] = __builtin_bit_cast(
                    float2v, __builtin_amdgcn_raw_buffer_load_b64(rml, (place * kPartMl + 2 * row) * 4, 0, kDeviceScope));
#pragma unroll
                for (int x = 0; x < kPasses; ++x)
                    part[u][x] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(ro, part_at(place, x), 0, kDeviceScope));
            }
            merge_batch<kBatch, true>(
                m_all, l_all, count - s0, [&](int u) __attribute__((always_inline)) { return state[u]; },
                [&](int u, PartWeights w) __attribute__((always_inline)) {
#pragma unroll
                    for (int x = 0; x < kPasses; ++x) sum[x] = merged(sum[x], part[u][x], w);
                });
        }
        store_rows(sum, l_all, mine.out);
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
    // (Of a score_scale of 0 the smallest number: a hidden token's -inf times it is still -inf; of
    // the largest a finite one, so that a score of 0 stays 0.)
    p.score_log2 = std::clamp(std::fabs(a.score_scale) * kLog2e, FLT_MIN, FLT_MAX);
    const std::int64_t items = static_cast<std::int64_t>(a.batch) * a.kv_heads * p.tiles;
    // Places of one of them, and its end rounded up to a range's length.
    const std::int64_t most = 2 * ((p.most_tokens - 1) / kCacheKeys + 1 + kSwitch);
    if (items > 0x3fffffffLL / most) return hipErrorInvalidConfiguration;
    int units = 0;
    const hipError_t found = check_device(&units);
    if (found != hipSuccess) return found;
    const int held = std::min(kRanges, groups_per_unit(p.group <= 8 ? 8 : 16) * units);
    p.ranges = static_cast<int>(std::min<std::int64_t>(held, (items * most - 1) / kLeastSteps + 1));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool bf16 = a.dtype == TILEMIX_DTYPE_BF16;
    const unsigned workgroups = static_cast<unsigned>(p.ranges);
    auto launch = [&](auto groups, auto rows) {
        constexpr int kGroups = decltype(groups)::value, kRows = decltype(rows)::value;
        if (bf16)
            cache4_attention_kernel<kGroups, true, kRows><<<workgroups, kThreads, 0, s>>>(p);
        else
            cache4_attention_kernel<kGroups, false, kRows><<<workgroups, kThreads, 0, s>>>(p);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Eight = std::integral_constant<int, 8>;
    using Sixteen = std::integral_constant<int, 16>;
    if (p.group <= 8)
        p.cache.groups == 1 ? launch(One{}, Eight{}) : launch(Two{}, Eight{});
    else
        p.cache.groups == 1 ? launch(One{}, Sixteen{}) : launch(Two{}, Sixteen{});
    return hipGetLastError();
}
