// Attention of packed sequences with grouped query heads for gfx950
// (tilemix_attention_packed): fp16 / bf16, causal with rows aligned at the end
// of their sequence's keys, or not causal.
//
// O[t, h] = sum_j p_j v[j, h / G],  p = softmax_j(scale q[t, h] . k[j, h / G]).
//
//  * A workgroup of four waves owns 32 query rows per wave: kTeam heads of one
//    key head (kTeam = the largest power of two up to 4 that divides G) x
//    128 / kTeam tokens. Waves of different heads with the same tokens share each
//    K / V tile and end at the same diagonal, so a causal walk has less masked
//    work than with 128 tokens of one head, and a short sequence fills its
//    workgroup.
//  * Which tokens a workgroup takes is found on the device (find_work), from the
//    lengths, blocks of more key tiles first: the host knows neither the lengths
//    nor the longest.
//  * Where the blocks are few, several workgroups walk a block's key tiles (kSplit).
//  * Scores, softmax and P.V as in attention_kernel (attention.hip): S^T = K Q^T
//    and O^T = V^T P^T on 32x32x16 MFMAs, probabilities kept in registers, K / V
//    tiles by LDS DMA.
//  * Every tile is addressed through a buffer that starts at its first row and ends
//    after the sequence's last, so rows of the next sequence read as zero and a
//    sequence may pass 2 GiB.
//
// Long walks are bound by the matrix unit at the power limit's clock beside the softmax's
// vector work: 16384 tokens, 32 heads (8 key heads) x 128, causal, bf16: 2.0 ms, 1.05
// PFLOP/s, matrix unit busy 57 % of cycles. Short ones by a block's start and end, about
// 10 us (queries, first tiles, O): 16 x 1024 tokens 182 to 235 us, 0.6 to 0.75 PFLOP/s;
// one of 250 tokens 6 us.

#include "attention_tiles.h"
#include "serving.h"
#include "tilemix_capi.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace tilemix {
namespace {

constexpr int kBlockShift = 7;
constexpr int kBlockRows = 1 << kBlockShift;  // query rows (tokens x heads) of a workgroup

struct PackedParams {
    const std::uint16_t* Q;
    const std::uint16_t* K;
    const std::uint16_t* V;
    std::uint16_t* O;
    const std::int32_t* q_starts;
    const std::int32_t* k_starts;
    std::int64_t q_row, k_row, v_row, o_row;      // elements between tokens
    std::int64_t q_head, k_head, v_head, o_head;  // and between heads
    int batch;
    int q_tokens, k_tokens;
    int kv_heads;
    int group;       // query heads per key head
    int chunks;      // group / team
    int team_shift;  // log2 of the heads of a workgroup
    int d;
    int causal;
    int negate;  // score_scale < 0: Q is negated
    float score_log2;  // |score_scale| log2(e)
    int longest_first;
    int places;        // workgroups of a team that share its blocks' key tiles; 0: one each
    // Of a split call: a workspace of the library.
    float* part_o;
    float* part_ml;
    unsigned* arrivals;
};

constexpr int kMostParts = 512;  // workgroups of a split call
constexpr int kLeastTiles = 4;   // key tiles of a split (8: 1 to 6 us more at 8 to 20 tiles a block)
constexpr int kSplitWalk = 12;   // a split call's average walk, in key tiles
static_assert(std::size_t{kMostParts} * kBlockRows * kMaxHeadDim <= kSplitScratchFloats &&
                  std::size_t{kMostParts} * kBlockRows * 2 <= kSplitStateFloats && kMostParts <= kSplitArrivals,
              "a split call's parts fit a workspace");

// ------------------------------------------------------------ work items

struct Sequence {
    int q0, q_len, k0, k_len;
};

// Bounds of sequence b, inside the tensors whatever the starts hold.
__device__ __forceinline__ Sequence sequence_at(const PackedParams& p, int b) {
    Sequence s;
    s.q0 = min(max(p.q_starts[b], 0), p.q_tokens);
    s.q_len = min(max(p.q_starts[b + 1], s.q0), p.q_tokens) - s.q0;
    s.k0 = min(max(p.k_starts[b], 0), p.k_tokens);
    s.k_len = min(max(p.k_starts[b + 1], s.k0), p.k_tokens) - s.k0;
    return s;
}

// Sum or maximum over the wave's lanes, in every lane (DPP steps as in wave_max_bits).
template <typename F>
__device__ __forceinline__ int wave_reduce(int v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false));
    int a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    v = f(a, b);
    a = v;
    b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return __builtin_amdgcn_readfirstlane(f(a, b));
}

// Blocks of 1 << shift query tokens of a sequence that walk at least `tiles` key tiles.
__device__ __forceinline__ int blocks_walking(const Sequence& s, int shift, int tiles, bool causal) {
    const int blocks = static_cast<int>((static_cast<unsigned>(s.q_len) + (1u << shift) - 1) >> shift);
    if (tiles <= 0) return blocks;
    // More than `hidden` keys are as many tiles; k_len and the rows are under 2^31, a tile count under 2^25.
    const unsigned hidden = static_cast<unsigned>(kTileKeys) * static_cast<unsigned>(tiles - 1);
    if (static_cast<unsigned>(s.k_len) <= hidden) return 0;
    if (!causal) return blocks;
    // Block j sees min(k_len, k_len - q_len + (j + 1 << shift)) keys: too few up to row `few`.
    const int few = s.q_len - static_cast<int>(static_cast<unsigned>(s.k_len) - hidden);
    return blocks - (max(few, 0) >> shift);
}

// What a workgroup does: a block of a sequence, and of its key tiles one of `splits` ranges.
struct Work {
    Sequence seq;
    int block;
    int slot;  // the block's number among all
    int split, splits;  // at most `splits` ranges of its key tiles; kSplit: which of them
};

// The work of place number `place` of a team, false past the last. kSplit: the team's
// `places` are dealt out to its blocks. Wave-uniform.
//
// Up to 64 sequences, one a lane: in order where all blocks start at once, else blocks of more
// key tiles first (the last to start are the shortest; a long walk that starts last would run
// alone), found by a search over tile counts. More sequences keep their order, as
// every step of that search would read all of their lengths (1000 sequences of 50 tokens, 32 heads: 707 us, 150 so;
// what the order costs: 100 of 200 tokens and one of 8192, 612 to 622 us with the long one first, 624 to 626 last): sequence b's blocks
// have the numbers from floor(start / tokens of a block) + b on, which leaves room for
// all of them, and is found by a search over the starts. Numbers left over have no work.
template <bool kSplit>
__device__ __forceinline__ bool find_work(const PackedParams& p, int place, int shift, int lane, Work& work) {
    auto divide = [&](int blocks) {
        work.splits = max(p.places / max(blocks, 1), 1);
        work.slot = kSplit ? place / work.splits : place;
        work.split = kSplit ? place - work.slot * work.splits : 0;
        return work.slot < blocks;
    };
    Sequence& found = work.seq;
    if (p.batch == 1) {
        found = sequence_at(p, 0);
        const int blocks = blocks_walking(found, shift, 0, false);
        if (!divide(blocks)) return false;
        work.block = blocks - 1 - work.slot;
        return true;
    }
    if (p.batch > kWave) {
        auto number_of = [&](int b) { return (min(max(p.q_starts[b], 0), p.q_tokens) >> shift) + b; };
        if (!divide(number_of(p.batch))) return false;
        int low = 0, count = p.batch;  // the last of these whose number is at most the slot
        for (int step = count; step > 1;) {
            step = (count + kWave - 1) / kWave;
            const bool reached = lane * step < count && number_of(low + lane * step) <= work.slot;
            const std::uint64_t those = __ballot(reached);
            if (!those) return false;  // rows before the first sequence
            const int last = (kWave - 1 - __builtin_clzll(those)) * step;
            low += last;
            count = min(count - last, step);
        }
        low = __builtin_amdgcn_readfirstlane(low);
        found = sequence_at(p, low);
        work.block = blocks_walking(found, shift, 0, false) - 1 - (work.slot - number_of(low));
        return work.block >= 0;
    }
    Sequence mine{0, 0, 0, 0};
    if (lane < p.batch) mine = sequence_at(p, lane);
    // Blocks that come before the slot: `above` of the lane's, and among `here` those of the lanes before.
    int above = 0, here = blocks_walking(mine, shift, 0, false);
    int before = static_cast<int>(prefix_sum(here));
    if (!divide(__builtin_amdgcn_readlane(before, kWave - 1))) return false;
    int rest = work.slot;
    if (p.longest_first) {
        const bool causal = p.causal != 0;
        auto sum = [](int v) { return wave_reduce(v, [](int a, int b) { return a + b; }); };
        // The most tiles of which more than `slot` blocks have as many.
        const unsigned keys = wave_reduce(mine.k_len, [](int a, int b) { return max(a, b); });
        int low = 0, high = static_cast<int>((keys + kTileKeys - 1) / kTileKeys) + 1;
        while (high - low > 1) {
            const int middle = (low + high) >> 1;
            if (sum(blocks_walking(mine, shift, middle, causal)) > work.slot)
                low = middle;
            else
                high = middle;
        }
        // Among the blocks of exactly `low` tiles.
        above = blocks_walking(mine, shift, low + 1, causal);
        here = blocks_walking(mine, shift, low, causal) - above;
        before = static_cast<int>(prefix_sum(here));
        rest -= sum(above);
    }
    const int at = __builtin_ctzll(__ballot(before > rest));
    found.q0 = __builtin_amdgcn_readlane(mine.q0, at);
    found.q_len = __builtin_amdgcn_readlane(mine.q_len, at);
    found.k0 = __builtin_amdgcn_readlane(mine.k0, at);
    found.k_len = __builtin_amdgcn_readlane(mine.k_len, at);
    // Blocks of a sequence walk more tiles the later they are.
    work.block = blocks_walking(found, shift, 0, false) - 1 - __builtin_amdgcn_readlane(above, at) -
                 (rest - __builtin_amdgcn_readlane(before - here, at));
    return true;
}

// ------------------------------------------------------- 16-bit arithmetic

template <bool kBf16>
__device__ __forceinline__ float16v mfma_32x32x16(uint4v a, uint4v b, float16v c) {
    if constexpr (kBf16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// sum + both halves of a pair.
template <bool kBf16>
__device__ __forceinline__ float add_pair(std::uint32_t pair, float sum) {
    if constexpr (kBf16)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2v, pair), bf2v{1.0f, 1.0f}, sum, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, pair), half2v{1.0f16, 1.0f16}, sum, false);
}

// softmax_tile of attention.hip for either type. The row sums take exactly the
// rounded probabilities that P.V uses: their rounding (2^-8 of each for bf16, 2^-11 for fp16)
// then cancels where values agree, and the rest is of the size of O's own rounding.
// For fp16 st.m lies 7 below the maximum, so that the largest probability is 2^7 and, as
// kLazyRescale is 8, none passes 2^15: half of fp16's least step is 2^-32 of the largest then,
// and many keys far below it keep their weight (700 of 2^-25.2 each were 0).
template <int kOB, bool kBf16>
__device__ __forceinline__ void softmax_rows(RowState<kOB>& st, const float16v (&x)[2], float c, uint4v (&p)[4]) {
    constexpr float kRaised = kBf16 ? 0.0f : 7.0f;
    static_assert(kBf16 || kRaised + kLazyRescale < 16.0f, "probabilities stay in fp16's range");
    const float largest = max3(block_max16(x[0]), block_max16(x[1]), block_max16(x[1]));
    const float tile = kBf16 ? largest * c : __builtin_fmaf(largest, c, -kRaised);  // c >= 0
    if (__any(tile > st.m + kLazyRescale)) {
        float a = tile, b = tile;
        permlane32_swap(a, b);
        const float m_new = fmaxf(st.m, max3(a, b, b));
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - m_new);
        st.m = m_new;
#pragma unroll
        for (int fb = 0; fb < kOB; ++fb) st.o[fb] *= alpha;
        st.lsum *= alpha;
    }
    const float neg_m = st.m == -INFINITY ? 0.0f : -st.m;
    float part[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        const int kb = ks >> 1, base = 8 * (ks & 1);
#pragma unroll
        for (int e = 0; e < 8; e += 2)
            p[ks][e / 2] = pack_pair<kBf16>(__builtin_amdgcn_exp2f(__builtin_fmaf(x[kb][base + e], c, neg_m)),
                                            __builtin_amdgcn_exp2f(__builtin_fmaf(x[kb][base + e + 1], c, neg_m)));
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = add_pair<kBf16>(p[ks][e], sum);
        part[ks] = sum;
        if (ks == 1) set_priority<2>();
    }
    st.lsum += (part[0] + part[1]) + (part[2] + part[3]);
}

// Whether any 16-bit value of the fragment is infinite or NaN.
template <bool kBf16>
__device__ __forceinline__ bool not_finite(uint4v v) {
    constexpr unsigned kExponent = kBf16 ? 0x7f80u : 0x7c00u;
    bool any = false;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        any |= (v[w] & kExponent) == kExponent || (v[w] & (kExponent << 16)) == (kExponent << 16);
    return any;
}

// 8-bit masks (bit e: half e) of the +inf, -inf and NaN values of a fragment, which become
// 0 in it.
template <bool kBf16>
__device__ __forceinline__ uint4v take_out_special(uint4v v, unsigned (&masks)[3]) {
    constexpr unsigned kExponent = kBf16 ? 0x7f80u : 0x7c00u;
    masks[0] = masks[1] = masks[2] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned x = (v[e / 2] >> (16 * (e % 2))) & 0xffffu, magnitude = x & 0x7fffu;
        if (magnitude >= kExponent) {
            const int kind = magnitude > kExponent ? 2 : static_cast<int>(x >> 15);
#pragma unroll
            for (int k = 0; k < 3; ++k) masks[k] |= (kind == k ? 1u : 0u) << e;
            v[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
        }
    }
    return v;
}

// How a block's key tiles are walked: in one piece; in ranges, each by a workgroup of its own,
// whose rows meet in the library's workspace, where the workgroup that arrives last
// merges them in order; in the same ranges by one workgroup, which merges them in the same order
// for the same bits (captured calls, which have no workspace).
enum class Walk { kWhole, kSplit, kInTurn };

template <int DC, bool kBf16, Walk kWalk>
__global__ __launch_bounds__(kThreadsPerGroup, 2) void packed_attention_kernel(const PackedParams p) {
    constexpr bool kSplit = kWalk == Walk::kSplit, kInTurn = kWalk == Walk::kInTurn;
    using L = Layout<DC>;
    constexpr int kDP = L::kDP;
    constexpr int kOB = DC;
    constexpr int kQC = kDP / 16;
    // K | V 0 | V 1
    __shared__ __attribute__((aligned(16))) unsigned char smem[L::kKBytes + 2 * L::kVBytes];
    __shared__ __attribute__((aligned(16))) unsigned char lds_spare[1024];  // landing area of the spare DMA slots
    // Which values of a diagonal tile are +inf, -inf and NaN, a byte for each 16-byte chunk; and
    // the last tile (counted from 1) that has any.
    constexpr int kChunks = kDP / 8;
    __shared__ __attribute__((aligned(16))) unsigned char lds_special[3][kTileKeys * kChunks];
    __shared__ int lds_special_tile;
    constexpr int kQuads = 4 * kOB;
    // kInTurn: O of the ranges so far, [quad][thread]. (Dynamic, as an array of known size would
    // have the compiler allocate accumulation registers for one workgroup a CU, which the softmax
    // pays for: 2 x 512 tokens after 7680 keys 245 us, when 195 so; now 169, in one piece 160.)
    extern __shared__ float4v lds_merged[];
    unsigned char* const lds_k = smem;
    unsigned char* const lds_v = smem + L::kKBytes;
    const unsigned lds_k_address = lds_address_of(smem);
    const unsigned lds_v_address = lds_k_address + L::kKBytes;
    const unsigned lds_spare_address = lds_address_of(lds_spare);

    const int tid = threadIdx.x;
    const int lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15;
    const int q = lane & 31;
    const int h = lane >> 5;
    const int d = p.d;

    // Consecutive workgroups go to consecutive XCDs: with eight key heads (or a
    // multiple) each XCD keeps the K / V of its own heads in its L2.
    const int teams = p.kv_heads * p.chunks;
    const int team = blockIdx.x % teams;
    const int kv_head = p.chunks == 1 ? team : team % p.kv_heads, chunk = p.chunks == 1 ? 0 : team / p.kv_heads;
    const int team_heads = 1 << p.team_shift;
    const int tokens = kBlockRows >> p.team_shift;
    Work work;
    if (!find_work<kSplit>(p, blockIdx.x / teams, kBlockShift - p.team_shift, lane, work)) return;
    const Sequence& seq = work.seq;
    const int context = seq.k_len - seq.q_len;  // row i sees keys up to context + i
    const int head = kv_head * p.group + (chunk << p.team_shift) + (wave & (team_heads - 1));
    const int t0 = work.block * tokens;
    const int tw = t0 + kRowsPerWave * (wave >> p.team_shift);  // the wave's first token

    // ---------------------------------------------------------------- Q
    uint4v qf[kQC];
    {
        const bool row_ok = tw + q < seq.q_len;
        const std::uint16_t* const row = p.Q + static_cast<std::int64_t>(seq.q0 + tw + q) * p.q_row + head * p.q_head;
#pragma unroll
        for (int c = 0; c < kQC; ++c) {
            const int feature = 16 * c + 8 * h;
            qf[c] = row_ok && feature < d ? *reinterpret_cast<const uint4v*>(row + feature) : uint4v{0u, 0u, 0u, 0u};
            if (p.negate) qf[c] ^= 0x80008000u;
        }
    }

    // ------------------------------------------------------ tile movement
    const int k_row_bytes = static_cast<int>(p.k_row * 2), v_row_bytes = static_cast<int>(p.v_row * 2);
    const std::uint16_t* const Ks = p.K + static_cast<std::int64_t>(seq.k0) * p.k_row + kv_head * p.k_head;
    const std::uint16_t* const Vs = p.V + static_cast<std::int64_t>(seq.k0) * p.v_row + kv_head * p.v_head;
    int off_k[L::kKPerWave], off_v[L::kVPerWave];
    unsigned dst_k[L::kKPerWave], dst_v[L::kVPerWave];
#pragma unroll
    for (int t = 0; t < L::kKPerWave; ++t) {
        const int w = wave + kWavesPerGroup * t;
        off_k[t] = w < L::kKLoads ? L::template kv_lane_offset<true>(w, lane, L::kKStride, 2 * d, k_row_bytes) : kOutOfRange;
        dst_k[t] = w < L::kKLoads ? lds_k_address + 1024 * w : lds_spare_address;
    }
#pragma unroll
    for (int t = 0; t < L::kVPerWave; ++t) {
        const int w = wave + kWavesPerGroup * t;
        off_v[t] = w < L::kVLoads ? L::template kv_lane_offset<false>(w, lane, L::kVStride, 2 * d, v_row_bytes) : kOutOfRange;
        dst_v[t] = w < L::kVLoads ? lds_v_address + 1024 * w : lds_spare_address;
    }
    // The rows of tile j that the sequence has, as a buffer (64 rows reach under 2 GiB).
    auto tile_rows = [&](const std::uint16_t* rows, std::int64_t row, int row_bytes, int j) {
        const int count = min(seq.k_len - j * kTileKeys, kTileKeys);
        return make_rsrc(rows + static_cast<std::int64_t>(j) * kTileKeys * row, (count - 1) * row_bytes + 2 * d);
    };
    auto issue_k = [&](int j) {
        const int4v r = tile_rows(Ks, p.k_row, k_row_bytes, j);
        if constexpr (L::kKLoads % kWavesPerGroup == 0) {
            load_slots(r, dst_k[0], off_k, 0);
        } else {
#pragma unroll
            for (int t = 0; t < L::kKPerWave; ++t) load_to_lds(r, dst_k[t], off_k[t], 0);
        }
    };
    auto issue_v = [&](int j, int buffer) {
        const int4v r = tile_rows(Vs, p.v_row, v_row_bytes, j);
        const unsigned shift = buffer ? static_cast<unsigned>(L::kVBytes) : 0u;
        if constexpr (L::kVLoads % kWavesPerGroup == 0) {
            load_slots(r, dst_v[0] + shift, off_v, 0);
        } else {
#pragma unroll
            for (int t = 0; t < L::kVPerWave; ++t)
                load_to_lds(r, dst_v[t] == lds_spare_address ? dst_v[t] : dst_v[t] + shift, off_v[t], 0);
        }
    };
    auto tile_barrier = [&]() {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // own tile loads: vmcnt(0)
        __syncthreads();
    };

    int k_lane[kQC], v_lane[kOB];
#pragma unroll
    for (int c = 0; c < kQC; ++c) k_lane[c] = L::k_at(q, 32 * c + 16 * h);
#pragma unroll
    for (int fb = 0; fb < kOB; ++fb)
        v_lane[fb] = L::v_at(4 * h + (i >> 2), 2 * (16 * fb + (kDP / 2) * ((lane >> 4) & 1) + 4 * (i & 3)));

    // ---------------------------------------------------------- key loop
    RowState<kOB> st;
#pragma unroll
    for (int fb = 0; fb < kOB; ++fb) st.o[fb] = float16v{};
    st.lsum = 0.0f;
    st.m = -INFINITY;

    // Last key that some row of the workgroup / of the wave sees, and all rows of the wave see.
    const int group_last = p.causal ? last_seen(context, t0 + tokens - 1, seq.q_len) : seq.k_len - 1;
    const int all_tiles = group_last < 0 ? 0 : group_last / kTileKeys + 1;
    // Ranges of at least kLeastTiles tiles (one, of none, of a block without keys). A tile takes
    // 1.3 us, and the last workgroup merges a part in 0.8 us (latency of 64 KB): of n tiles,
    // sqrt(1.6 n) ranges are soonest done (one token of 30000 keys, 8 key heads: 64 ranges 74 us,
    // 27 54 us).
    const int splits =
        kWalk == Walk::kWhole ? 1 : min(work.splits, max(min(all_tiles / kLeastTiles, static_cast<int>(sqrtf(1.6f * all_tiles))), 1));
    if (kSplit && work.split >= splits) return;
    auto range_start = [&](int split) { return split * (all_tiles / splits) + min(split, all_tiles % splits); };
    const int first_tile = kSplit ? range_start(work.split) : 0;
    const int tiles = kSplit ? range_start(work.split + 1) : all_tiles;
    const int wave_last = tw >= seq.q_len ? -1 : p.causal ? last_seen(context, tw + kRowsPerWave - 1, seq.q_len) : seq.k_len - 1;
    const int all_last = p.causal ? last_seen(context, tw, seq.q_len) : seq.k_len - 1;

    // A row's probability of a key that it does not see is 0, but 0 times an infinite or NaN
    // value is NaN: such values are taken out of diagonal tiles, and put into the rows that
    // see them afterwards.
    const int first_hidden = p.causal ? context + t0 + 1 : seq.k_len;  // first key that some row of the workgroup does not see
    if (tid == 0) lds_special_tile = 0;
    int v_buffer = 0;
    // kInTurn: the range under way, and the merged rows' states.
    int range = 0, range_end = range_start(1);
    float merged_m = -INFINITY, merged_l = 0.0f;
    auto row_sum = [&]() __attribute__((always_inline)) {
        float a = st.lsum, b = st.lsum;
        permlane32_swap(a, b);
        return a + b;
    };
    if (tiles > first_tile) {
        issue_k(first_tile);
        issue_v(first_tile, 0);
    }
    for (int j = first_tile; j < tiles; ++j) {
        const int k0 = j * kTileKeys;
        tile_barrier();  // K_j, V_j landed; every wave finished P.V of the previous tile
        set_priority<2>();
        const bool active = k0 <= wave_last;
        // (Compared without k0 + kTileKeys, which may be 2^31.)
        const bool masked = k0 > min(all_last, seq.k_len - 1) - (kTileKeys - 1);
        float16v s[2];
        float c = p.score_log2;
        if (active) {
            s[0] = float16v{};
            s[1] = float16v{};
            uint4v kf[3][2];
            auto load_c = [&](int cc, uint4v (&dst)[2]) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    dst[kb] = *reinterpret_cast<const uint4v*>(lds_k + 32 * L::kKStride * kb + k_lane[cc]);
            };
            load_c(0, kf[0]);
            load_c(1, kf[1]);
#pragma unroll
            for (int cc = 0; cc < kQC; ++cc) {
                if (cc + 2 < kQC) load_c(cc + 2, kf[(cc + 2) % 3]);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) s[kb] = mfma_32x32x16<kBf16>(kf[cc % 3][kb], qf[cc], s[kb]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // The last key that the lane's row sees, from the tile's first key of the lane.
        // (last_seen of row tw + q, the wave's part of it a scalar.)
        int seen = (p.causal ? context + tw + min(q, seq.q_len - 1 - tw) : seq.k_len - 1) - k0 - 4 * h;
        if (active && masked) {
            asm volatile("" : "+v"(seen));
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[kb][e] = 32 * kb + 8 * (e >> 2) + (e & 3) > seen ? -INFINITY : s[kb][e] * c;
            c = 1.0f;
        }
        const bool diagonal = k0 >= first_hidden - (kTileKeys - 1);  // of the workgroup
        unsigned char* const v_tile = lds_v + (v_buffer ? L::kVBytes : 0);
        constexpr int kChecks = kTileKeys * kChunks / kThreadsPerGroup;  // chunks of a thread
        auto checked = [&](int x) {
            const int id = x * kThreadsPerGroup + tid;
            return reinterpret_cast<uint4v*>(v_tile + L::v_at(id / kChunks, 16 * (id % kChunks)));
        };
        if (p.causal && diagonal) {
            bool special = false;
#pragma unroll
            for (int x = 0; x < kChecks; ++x) special |= not_finite<kBf16>(*checked(x));
            if (special) lds_special_tile = j + 1;
        }
        tile_barrier();  // every wave finished reading K_j (and P.V of the previous tile)
        set_priority<0>();
        const bool special = p.causal && diagonal && lds_special_tile == j + 1;
        if (special) {
#pragma unroll 1
            for (int x = 0; x < kChecks; ++x) {
                unsigned masks[3];
                const uint4v clean = take_out_special<kBf16>(*checked(x), masks);
                *checked(x) = clean;
#pragma unroll
                for (int kind = 0; kind < 3; ++kind)
                    lds_special[kind][x * kThreadsPerGroup + tid] = static_cast<unsigned char>(masks[kind]);
            }
            __syncthreads();
        }
        if (j + 1 < tiles) {
            issue_k(j + 1);
            issue_v(j + 1, v_buffer ^ 1);
        }
        if (active) {
            uint4v ph[4];
            softmax_rows<kOB, kBf16>(st, s, c, ph);
            // V^T fragment of step t = (key step t / kOB, feature block t % kOB).
            auto v_frag = [&](int t) {
                const unsigned char* const lo = v_tile + 16 * L::kVStride * (t / kOB) + v_lane[t % kOB];
                return __builtin_bit_cast(uint4v, concat(read_tr16(lo), read_tr16(lo + 8 * L::kVStride)));
            };
            constexpr int kSteps = 4 * kOB;
            constexpr int kAhead = 3;
            set_priority<0>();
            uint4v vf[kAhead + 1];
#pragma unroll
            for (int t = 0; t < kAhead; ++t)
                if (t < kSteps) vf[t] = v_frag(t);
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                if (t + kAhead < kSteps) vf[(t + kAhead) % (kAhead + 1)] = v_frag(t + kAhead);
                st.o[t % kOB] = mfma_32x32x16<kBf16>(vf[t % (kAhead + 1)], ph[t / kOB], st.o[t % kOB]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (special) {
#pragma unroll 1
                for (int kind = 0; kind < 3; ++kind) {
                    unsigned seen_bits[kChunks / 4] = {};  // features in which the row sees such a value
#pragma unroll 1
                    for (int key = 0; key < kTileKeys; ++key) {
                        const auto* const bits = reinterpret_cast<const unsigned*>(lds_special[kind] + key * kChunks);
#pragma unroll
                        for (int x = 0; x < kChunks / 4; ++x)
                            if (key <= seen + 4 * h) seen_bits[x] |= bits[x];
                    }
                    const float value = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
#pragma unroll
                    for (int fb = 0; fb < kOB; ++fb)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int feature = (e < 8 ? 0 : kDP / 2 - 16) + 16 * fb + 8 * (e / 4) + e % 4;  // + 4 h
                            st.o[fb][e] += (seen_bits[feature / 32] >> (feature % 32 + 4 * h)) & 1u ? value : 0.0f;
                        }
                }
            }
        }
        v_buffer ^= 1;
        if (kInTurn && splits > 1 && j + 1 == range_end) {
            const PartWeights w = merge_part(merged_m, merged_l, st.m, row_sum());
#pragma unroll
            for (int x = 0; x < kQuads; ++x) {
                float4v& all = lds_merged[x * kThreadsPerGroup + tid];
                const float16v& o = st.o[x / 4];
                const int e = 4 * (x % 4);
                all = merged(range == 0 ? float4v{0.0f, 0.0f, 0.0f, 0.0f} : all, float4v{o[e], o[e + 1], o[e + 2], o[e + 3]}, w);
            }
#pragma unroll
            for (int fb = 0; fb < kOB; ++fb) st.o[fb] = float16v{};
            st.lsum = 0.0f;
            st.m = -INFINITY;
            range_end = range_start(++range + 1);
        }
    }

    // ---------------------------------------------------------- epilogue
    float l = row_sum();
    if constexpr (kInTurn) {
        if (splits > 1) {
            l = merged_l;
#pragma unroll
            for (int x = 0; x < kQuads; ++x) {
                const float4v all = lds_merged[x * kThreadsPerGroup + tid];
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[x / 4][4 * (x % 4) + e] = all[e];
            }
        }
    }
    if constexpr (kSplit) {
        if (splits > 1) {
            // Parts: [item][split], O as the threads hold it, and (m, l) of the 128 rows.
            const int item = work.slot * teams + team, row = kRowsPerWave * wave + q;
            const std::int64_t parts = gridDim.x;
            const auto ro = shared_rows(p.part_o, parts * kQuads * kThreadsPerGroup * 4);
            const auto rml = shared_rows(p.part_ml, parts * kBlockRows * 2);
            auto o_at = [&](int part, int x) { return ((part * kQuads + x) * kThreadsPerGroup + tid) * 16; };
            auto ml_at = [&](int part) { return (part * kBlockRows + row) * 8; };
            const int first = item * work.splits;
#pragma unroll
            for (int x = 0; x < kQuads; ++x) {
                const float16v& o = st.o[x / 4];
                const int e = 4 * (x % 4);
                __builtin_amdgcn_raw_buffer_store_b128(
                    __builtin_bit_cast(uint4v, float4v{o[e], o[e + 1], o[e + 2], o[e + 3]}), ro, o_at(first + work.split, x), 0, kDeviceScope);
            }
            if (h == 0)
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uint2v, float2v{st.m, l}), rml, ml_at(first + work.split), 0,
                                                      kDeviceScope);
            if (!last_arrival(p.arrivals + item, splits, &lds_special_tile)) return;
            float m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int fb = 0; fb < kOB; ++fb) st.o[fb] = float16v{};
#pragma unroll 1
            for (int s = 0; s < splits; ++s) {
                const float2v state = __builtin_bit_cast(float2v, __builtin_amdgcn_raw_buffer_load_b64(rml, ml_at(first + s), 0, kDeviceScope));
                float4v part[kQuads];
#pragma unroll
                for (int x = 0; x < kQuads; ++x)
                    part[x] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(ro, o_at(first + s, x), 0, kDeviceScope));
                const PartWeights w = merge_part(m, l, state[0], state[1]);
#pragma unroll
                for (int x = 0; x < kQuads; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[x / 4][4 * (x % 4) + e] = merged(st.o[x / 4][4 * (x % 4) + e], part[x][e], w);
            }
        }
    }
    // 0: no key; NaN scores leave l NaN, and the row becomes NaN.
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    // Rows leave through LDS as whole lines: stored from registers, an instruction writes 16
    // bytes of each of 32 rows, and twice the bytes went to memory (16 x 1024 tokens, 32
    // heads x 128: 262 MB for 134, 250 us; 227 so). The wave's region lies in the K
    // tile or the V buffer that the last tile did not use: every wave has passed the last tile's
    // second barrier, so none reads them. 16-byte chunk c of a row lies at chunk
    // position (c + row) mod kChunks.
    static_assert(L::kKBytes >= 2 * kRowsPerWave * kDP * 2 && L::kVBytes >= 2 * kRowsPerWave * kDP * 2, "two waves' rows fit a tile");
    unsigned char* const region =
        (wave < 2 ? lds_k : lds_v + (v_buffer ? L::kVBytes : 0)) + (wave & 1) * kRowsPerWave * kDP * 2;
    auto chunk_at = [&](int row, int c) { return region + (row * kChunks + (c + row) % kChunks) * 16; };
#pragma unroll
    for (int fb = 0; fb < kOB; ++fb)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int feature = (r4 < 2 ? 0 : kDP / 2 - 16) + 16 * fb + 8 * r4;  // + 4 h
            const float4v value{st.o[fb][4 * r4], st.o[fb][4 * r4 + 1], st.o[fb][4 * r4 + 2], st.o[fb][4 * r4 + 3]};
            *reinterpret_cast<uint2v*>(chunk_at(q, feature / 8) + 8 * h) =
                uint2v{pack_pair<kBf16>(value[0] * inverse, value[1] * inverse),
                       pack_pair<kBf16>(value[2] * inverse, value[3] * inverse)};
        }
    std::uint16_t* const out = p.O + static_cast<std::int64_t>(seq.q0 + tw) * p.o_row + head * p.o_head;
    constexpr int kStores = kRowsPerWave * kChunks / kWave;
    uint4v piece[kStores];
#pragma unroll
    for (int x = 0; x < kStores; ++x) {
        const int id = x * kWave + lane;
        piece[x] = *reinterpret_cast<const uint4v*>(chunk_at(id / kChunks, id % kChunks));
    }
#pragma unroll
    for (int x = 0; x < kStores; ++x) {
        const int id = x * kWave + lane, row = id / kChunks, c = id % kChunks;
        if (tw + row < seq.q_len && 8 * c < d)
            __builtin_nontemporal_store(piece[x], reinterpret_cast<uint4v_dword*>(out + row * p.o_row + 8 * c));
    }
}

template <int DC, Walk kWalk>
void launch_packed(const PackedParams& p, bool bf16, unsigned grid, hipStream_t stream) {
    constexpr std::size_t kMerged = kWalk == Walk::kInTurn ? std::size_t{kBlockRows} * 32 * DC * sizeof(float) : 0;
    if (bf16)
        packed_attention_kernel<DC, true, kWalk><<<grid, kThreadsPerGroup, kMerged, stream>>>(p);
    else
        packed_attention_kernel<DC, false, kWalk><<<grid, kThreadsPerGroup, kMerged, stream>>>(p);
}

template <Walk kWalk>
hipError_t launch_packed(const PackedParams& p, bool bf16, std::int64_t workgroups, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(workgroups);
    switch ((p.d + 31) / 32) {
        case 1: launch_packed<1, kWalk>(p, bf16, grid, stream); break;
        case 2: launch_packed<2, kWalk>(p, bf16, grid, stream); break;
        case 3: launch_packed<3, kWalk>(p, bf16, grid, stream); break;
        default: launch_packed<4, kWalk>(p, bf16, grid, stream); break;
    }
    return hipGetLastError();
}

struct SplitCall {
    PackedParams p;
    bool bf16;
    std::int64_t grid;
    hipStream_t stream;
};

}  // namespace
}  // namespace tilemix

extern "C" int tilemix_attention_packed(const TileMixPackedAttentionArgs* args, void* stream) {
    using namespace tilemix;
    if (!args) return hipErrorInvalidValue;
    const TileMixPackedAttentionArgs& a = *args;
    if (a.batch < 0 || a.q_tokens < 0 || a.k_tokens < 0 || a.q_heads <= 0 || a.kv_heads <= 0 || a.d <= 0 ||
        a.q_heads % a.kv_heads != 0 || !std::isfinite(a.score_scale) ||
        (a.dtype != TILEMIX_DTYPE_F16 && a.dtype != TILEMIX_DTYPE_BF16))
        return hipErrorInvalidValue;
    if (a.d > kMaxHeadDim) return hipErrorNotSupported;
    if (a.d % 8 != 0) return hipErrorInvalidValue;
    PackedParams p{};
    Rows q, k, v, o;
    if (!make_rows(q, a.Q, a.q_tokens, a.q_heads, a.d, a.q_row_stride, a.q_head_stride, 8) ||
        !make_rows(k, a.K, a.k_tokens, a.kv_heads, a.d, a.k_row_stride, a.k_head_stride, 8) ||
        !make_rows(v, a.V, a.k_tokens, a.kv_heads, a.d, a.v_row_stride, a.v_head_stride, 8) ||
        !make_rows(o, a.O, a.q_tokens, a.q_heads, a.d, a.o_row_stride, a.o_head_stride, 4))
        return hipErrorInvalidValue;
    // A tile's rows are reached by 32-bit offsets.
    constexpr std::int64_t kReach = (std::int64_t{1} << 30) / kTileKeys;
    if (k.row > kReach || v.row > kReach) return hipErrorNotSupported;
    if (a.batch == 0 || a.q_tokens == 0) return hipSuccess;
    if (!a.q_starts) return hipErrorInvalidValue;
    p.Q = a.Q;
    p.K = a.K;
    p.V = a.V;
    p.O = a.O;
    p.q_starts = a.q_starts;
    p.k_starts = a.k_starts ? a.k_starts : a.q_starts;
    p.q_row = q.row, p.q_head = q.head;
    p.k_row = k.row, p.k_head = k.head;
    p.v_row = v.row, p.v_head = v.head;
    p.o_row = o.row, p.o_head = o.head;
    p.batch = a.batch;
    p.q_tokens = a.q_tokens;
    p.k_tokens = a.k_tokens;
    p.kv_heads = a.kv_heads;
    p.group = a.q_heads / a.kv_heads;
    p.team_shift = p.group % 4 == 0 ? 2 : p.group % 2 == 0 ? 1 : 0;
    p.chunks = p.group >> p.team_shift;
    p.d = a.d;
    p.causal = a.causal != 0;
    p.negate = a.score_scale < 0.0f;
    p.score_log2 = std::min(std::fabs(a.score_scale) * kLog2e, FLT_MAX);  // finite: a score of 0 stays 0
    // Blocks of all sequences: each has at most one that is not full (find_work: and, of many, one number).
    const int tokens = kBlockRows >> p.team_shift;
    const std::int64_t blocks = a.q_tokens / tokens + static_cast<std::int64_t>(a.batch > kWave ? a.batch : std::min(a.batch, a.q_tokens));
    const std::int64_t grid = blocks * p.kv_heads * p.chunks;
    if (grid > 0xffffffffLL / kThreadsPerGroup) return hipErrorInvalidConfiguration;  // threads of a launch
    int units = 0;
    const hipError_t found = check_device(&units);
    if (found != hipSuccess) return found;
    const bool bf16 = a.dtype == TILEMIX_DTYPE_BF16;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    // The order matters to more than one round of workgroups (4 x 2048 tokens, 16 heads x 64: in
    // order 59 us, longest first 52), the search's time to the rest (4 x 250: 8.7 us with it, 8.0).
    p.longest_first = grid > 2 * units;
    // Few blocks with long walks are split, into as many workgroups as are resident at
    // once. The lengths are not known here, so the average walk decides (2 x 256 tokens, 16 heads
    // x 128; in one piece and split): 6 tiles 17.7 and 19.8 us, 10 22.9 and 23.1, 18 33.6 and
    // 26.0, 34 52 and 34, 122 154 and 58; 2 x 512 tokens after 7680 keys 168 and 85.
    const std::int64_t teams = static_cast<std::int64_t>(p.kv_heads) * p.chunks, places = std::min(kMostParts, 2 * units) / teams;
    const double rows = static_cast<double>(a.q_tokens) / a.batch, keys = static_cast<double>(a.k_tokens) / a.batch;
    const double walk = (p.causal ? keys - 0.5 * std::min(rows, keys) : keys) / kTileKeys;
    if (blocks <= places && 2 * ((rows + tokens - 1) / tokens) * a.batch <= static_cast<double>(places) && walk >= kSplitWalk) {
        p.places = static_cast<int>(places);
        p.longest_first = 0;
        SplitCall call{p, bf16, places * teams, s};
        bool given = false;
        const hipError_t status = call_with_workspace(
            s,
            [](void* context, float* scratch, float* states, unsigned* arrivals) {
                SplitCall& c = *static_cast<SplitCall*>(context);
                c.p.part_o = scratch;
                c.p.part_ml = states;
                c.p.arrivals = arrivals;
                return launch_packed<Walk::kSplit>(c.p, c.bf16, c.grid, c.stream);
            },
            &call, given);
        if (given || status != hipSuccess) return status;
        return launch_packed<Walk::kInTurn>(p, bf16, grid, s);
    }
    return launch_packed<Walk::kWhole>(p, bf16, grid, s);
}
