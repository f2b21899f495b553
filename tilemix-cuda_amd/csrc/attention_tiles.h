#pragma once
// Tiles of the MFMA attention kernels (attention.hip, packed_attention.hip):
// LDS layout of K / V / K8 tiles, their LDS DMA, and the state of a wave's rows.

#include "attention_common.h"

namespace tilemix {
namespace {

constexpr int kThreadsPerGroup = 256;
constexpr int kWavesPerGroup = kThreadsPerGroup / kWave;
constexpr int kRowsPerWave = 32;

template <int DC>
struct Layout {
    static constexpr int kDP = 32 * DC;            // padded head dim, fp16 path
    static constexpr int kD8C = (DC + 1) / 2;      // 64-feature chunks, int8 path
    static constexpr int kDP8 = 64 * kD8C;
    // K / V rows hold 2 * kDP bytes. Rows of 256 bytes (d > 96) and 128 bytes
    // (32 < d <= 64) are unpadded, with 16-byte chunk c of row r at chunk
    // position (c + rot(r)) mod (chunks per row), so that the fragment reads
    // are free of LDS bank conflicts with no pad bytes to move (rot below).
    // Other rows are padded by 16 (K) or 32 (V) bytes. K8 rows are 128 bytes
    // (d > 64) or 64 bytes, rotated the same way.
    static constexpr int kRowBytes = kDP * 2;
    static constexpr bool kRotate = kRowBytes == 256 || kRowBytes == 128;
    static constexpr bool kRotate8 = kDP8 == 128 || kDP8 == 64;
    static constexpr int kKStride = kRotate ? kRowBytes : kRowBytes + 16;
    static constexpr int kVStride = kRotate ? kRowBytes : kRowBytes + 32;
    static constexpr int kK8Stride = kRotate8 ? kDP8 : kDP8 + 16;
    static constexpr int kKBytes = kTileKeys * kKStride;
    static constexpr int kVBytes = kTileKeys * kVStride;
    static constexpr int kK8Bytes = kTileKeys * kK8Stride;
    // One buffer_load ... lds per wave moves 1 KiB (64 lanes x 16 bytes).
    static constexpr int kKLoads = kKBytes / 1024;
    static constexpr int kVLoads = kVBytes / 1024;
    static constexpr int kK8Loads = kK8Bytes / 1024;
    static constexpr int kKPerWave = (kKLoads + kWavesPerGroup - 1) / kWavesPerGroup;
    static constexpr int kVPerWave = (kVLoads + kWavesPerGroup - 1) / kWavesPerGroup;
    static constexpr int kK8PerWave = (kK8Loads + kWavesPerGroup - 1) / kWavesPerGroup;
    // K, V buffer 0, K8, V buffer 1.
    static constexpr int kV1Offset = kVBytes + kK8Bytes;  // V buffer 1 - V buffer 0
    static constexpr int kSmemBytes = kKBytes + kVBytes + kK8Bytes + kVBytes;
    static_assert(kKBytes % 1024 == 0 && kVBytes % 1024 == 0 && kK8Bytes % 1024 == 0,
                  "tiles are whole wave loads");
    // Chunk rotation of a rotated row of kChunks 16-byte chunks. Key rows
    // (K, K8) are read as 32 consecutive rows x one chunk per half-wave: the
    // rows that share one 256-byte sweep of the banks share a rotation, and
    // consecutive sweeps step it by one chunk (measured on 64-byte K8 rows:
    // 13 % of LDS-active cycles in bank conflicts with a rotation that steps
    // every two rows, 0.9 % with this one). Value rows are read by
    // ds_read_b64_tr_b16 in 4-row x 16-feature blocks.
    template <int kChunks, bool kKey>
    __device__ static int rot(int row) {
        static_assert(kChunks == 16 || kChunks == 8 || kChunks == 4, "rotated rows are 256, 128 or 64 bytes");
        if constexpr (kKey)
            return kChunks == 16 ? row & 15 : kChunks == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
        else
            return kChunks == 16 ? (2 * row) & 15 : kChunks == 8 ? row & 6 : 2 * ((row >> 2) & 1);
    }
    // Offset of byte `byte` of row `row` in a rotated tile.
    template <int kChunks, bool kKey>
    __device__ static int rotated(int row, int byte) {
        return row * 16 * kChunks + ((((byte >> 4) + rot<kChunks, kKey>(row)) & (kChunks - 1)) << 4) + (byte & 15);
    }
    // Global offset that DMA lane `lane` of 1 KiB piece w fetches for a
    // rotated tile (kOutOfRange past the row's bytes): the inverse of rotated.
    template <int kChunks, bool kKey>
    __device__ static int rotated_lane(int w, int lane, int row_bytes, int global_row_bytes) {
        const int landing = 1024 * w + 16 * lane;
        const int row = landing / (16 * kChunks);
        const int column = ((((landing >> 4) & (kChunks - 1)) - rot<kChunks, kKey>(row)) & (kChunks - 1)) << 4;
        return column < row_bytes ? row * global_row_bytes + column : kOutOfRange;
    }
    // Offset of byte `byte` (< 2 * kDP, or < kDP8 for K8) of row `row` in the
    // K / V / K8 tile.
    __device__ static int k_at(int row, int byte) {
        if constexpr (kRotate) return rotated<kRowBytes / 16, true>(row, byte);
        else return row * kKStride + byte;
    }
    __device__ static int v_at(int row, int byte) {
        if constexpr (kRotate) return rotated<kRowBytes / 16, false>(row, byte);
        else return row * kVStride + byte;
    }
    __device__ static int k8_at(int row, int byte) {
        if constexpr (kRotate8) return rotated<kDP8 / 16, true>(row, byte);
        else return row * kK8Stride + byte;
    }
    // Global offset that DMA lane `lane` of 1 KiB piece w fetches.
    template <bool kKey>
    __device__ static int kv_lane_offset(int w, int lane, int stride, int row_bytes, int global_row_bytes) {
        if constexpr (kRotate) return rotated_lane<kRowBytes / 16, kKey>(w, lane, row_bytes, global_row_bytes);
        else return lane_offset(w, lane, stride, row_bytes, global_row_bytes);
    }
    __device__ static int k8_lane_offset(int w, int lane, int row_bytes) {
        if constexpr (kRotate8) return rotated_lane<kDP8 / 16, true>(w, lane, row_bytes, row_bytes);
        else return lane_offset(w, lane, kK8Stride, row_bytes, row_bytes);
    }
};

typedef float float16v __attribute__((ext_vector_type(16)));
typedef int int16v __attribute__((ext_vector_type(16)));

// Online-softmax state of the query row a lane owns (row lane & 31 of the
// wave's 32; lanes l and l ^ 32 hold the same row, each for half of every
// 32-key block), scores in the log2 domain, m raised lazily (kLazyRescale).
template <int kOB>
struct RowState {
    // O^T accumulators: o[fb][j] is output row R = 8 (j / 4) + 4 h + j % 4
    // (h = lane / 32) of feature block fb, i.e. feature 16 fb + R for R < 16
    // and kDP / 2 + 16 fb + R - 16 above (the two 16-row halves of a block
    // sit kDP / 2 features apart, which keeps the transposed V reads free of
    // bank conflicts).
    float16v o[kOB];
    float lsum;       // this lane's part of the row sum of P (the fp16 values P.V uses)
    float m;
};

// Maximum of the 16 values of a 32x32 accumulator block, 8 v_max3.
[[maybe_unused]] __device__ __forceinline__ float block_max16(const float16v& x) {
    const float a = max3(x[0], x[1], x[2]), b = max3(x[3], x[4], x[5]), e = max3(x[6], x[7], x[8]);
    const float f = max3(x[9], x[10], x[11]), g = max3(x[12], x[13], x[14]);
    return max3(max3(a, b, e), max3(f, g, x[15]), x[15]);
}

// load_to_lds with M0 = lds_address + kOffset, the add issued inside the asm
// so that the compiler keeps one scalar address per buffer, not one per slot.
template <int kOffset>
__device__ __forceinline__ void load_to_lds_at(int4v rsrc, unsigned lds_address, int voffset, int soffset) {
    if constexpr (kOffset == 0) {
        load_to_lds(rsrc, lds_address, voffset, soffset);
    } else {
        asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :
                     : "s"(lds_address), "v"(voffset), "s"(rsrc), "s"(soffset), "i"(kOffset)
                     : "memory", "scc");
    }
}

// The 1 KiB pieces one wave moves of a tile buffer that splits evenly over
// the workgroup's four waves: slot t lands 4 KiB past slot t - 1 (pieces
// wave, wave + 4, ...), so all slots share the first one's LDS address.
template <int t, int kSlots>
__device__ __forceinline__ void load_slots_from(int4v rsrc, unsigned first, const int (&voffset)[kSlots], int soffset) {
    if constexpr (t < kSlots) {
        load_to_lds_at<4096 * t>(rsrc, first, voffset[t], soffset);
        load_slots_from<t + 1, kSlots>(rsrc, first, voffset, soffset);
    }
}
template <int kSlots>
__device__ __forceinline__ void load_slots(int4v rsrc, unsigned first, const int (&voffset)[kSlots], int soffset) {
    load_slots_from<0, kSlots>(rsrc, first, voffset, soffset);
}

// The pieces one of eight waves moves of a tile buffer kBase bytes past the
// wave's first LDS address: slot t lands 8 KiB past slot t - 1. `base` bytes
// are added to the lanes' offsets, so the range check covers the whole address.
template <int kBase, int t, int kSlots>
__device__ __forceinline__ void load_slots_at(int4v rsrc, unsigned first, const int (&voffset)[kSlots], int base) {
    if constexpr (t < kSlots) {
        load_to_lds_at<kBase + 8192 * t>(rsrc, first, voffset[t] + base, 0);
        load_slots_at<kBase, t + 1, kSlots>(rsrc, first, voffset, base);
    }
}

}  // namespace
}  // namespace tilemix
