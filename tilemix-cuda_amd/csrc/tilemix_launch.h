#pragma once
// Host-side declarations shared by the TileMix translation units.

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace tilemix {

inline constexpr int kMaxHeadDim = 128;  // kFusedMaxHeadDim
inline constexpr int kQBlockRows = 128;  // kTileMixQQuantRows
inline constexpr int kKBlockRows = 64;   // kTileMixKQuantRows
inline constexpr int kCellRows = 16;     // kBlockM: routing cell height
inline constexpr int kCellKeys = 32;     // kBlockN: routing cell width

// One side (Q or K) of a quantizer launch. Inputs of head h start at
// x + h * in_head_stride, rows in_row_stride elements apart; outputs are
// contiguous per head.
struct QuantSide {
    const std::uint16_t* x;
    std::int8_t* x8;
    std::uint16_t* scales;
    std::int64_t in_head_stride;
    std::int64_t in_row_stride;
    int rows;
    int block_rows;
    int blocks;  // quantization blocks per head, 0 = side absent
};

// A [heads][rows][d] view, strides in elements, whose heads do not overlap:
// rows are at least d apart, and heads either follow one another (each head
// fits below the next head's start) or interleave inside every row (all
// heads' d elements fit in one row stride, e.g. a [rows][heads][d] tensor).
inline bool strided_heads_ok(int heads, int rows, int d, std::int64_t head_stride, std::int64_t row_stride) {
    if (row_stride < d) return false;
    if (heads <= 1) return true;
    const std::int64_t extent = static_cast<std::int64_t>(rows - 1) * row_stride + d;
    if (head_stride >= extent) return true;
    return head_stride >= d && static_cast<std::int64_t>(heads - 1) * head_stride + d <= row_stride;
}

// Whether the current device is one the kernels run on (hipErrorNotSupported
// otherwise), and its compute units.
hipError_t check_device(int* compute_units = nullptr);

// One of the library's split workspaces (attention.hip): floats of partial rows,
// floats of their states, arrival counters that are zero between launches.
inline constexpr std::size_t kSplitScratchFloats = std::size_t{8} << 20;  // 32 MiB
inline constexpr std::size_t kSplitStateFloats = std::size_t{128} << 10;  // 512 KiB
inline constexpr std::size_t kSplitArrivals = 1024;
using WorkspaceLaunch = hipError_t (*)(void* context, float* scratch, float* states, unsigned* arrivals);
// Calls launch(context, ...), which enqueues kernels on `stream` that use a workspace, ordered
// before and after what else uses it. given: false, and nothing is called, where `stream` is
// being captured (or the device has no workspace).
hipError_t call_with_workspace(hipStream_t stream, WorkspaceLaunch launch, void* context, bool& given);

QuantSide make_quant_side(const std::uint16_t* x, std::int8_t* x8, std::uint16_t* scales,
                          std::int64_t head_stride, int rows, int block_rows, std::int64_t row_stride);

hipError_t launch_quantize(const QuantSide& q, const QuantSide& k, int heads, int d,
                           hipStream_t stream);

}  // namespace tilemix
