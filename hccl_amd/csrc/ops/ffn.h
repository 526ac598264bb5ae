// Launch interface of the experts' feed-forward kernels (ffn_launch.h, instantiated per type in ffn_bf16.hip and ffn_f16.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hcclx {

constexpr uint32_t kFfnRanks = 64;

// The rows of the ranks, and the products' sizes.  Buffers of the plan hold the rows of all ranks back to back ("packed").
struct FfnRows {
    const uint64_t *counts;   // nullptr: capacity rows each
    uint32_t per_rank;
    uint32_t unit;
    uint32_t n;
    uint32_t capacity;
    uint32_t most;            // rows in all ranks together
    uint32_t dim;
    uint32_t hidden;
};

// The five products.  p: what a kernel needs of each rank, in this order.
enum FfnKind {
    kFfnGateUp,       // x, w_gate, w_up                        -> h, saved
    kFfnDown,         // w_down, out                       h    -> out
    kFfnGradHidden,   // dy, w_down                        saved -> h, dproj
    kFfnGradInput,    // w_gate, w_up, dx                  dproj -> dx
    kFfnGradWeights,  // x, dy, dw_gate, dw_up, dw_down    h, dproj -> dw_*
};
struct FfnArgs {
    FfnRows rows;
    const char *p[5][kFfnRanks];
    char *h;        // packed rows of `hidden` elements
    char *dproj;    // packed rows of 2 x `hidden` elements: gradients of both products of the forward pass
    float *saved;   // packed rows of 2 x `hidden` floats: both products of the forward pass; may be nullptr (kFfnGateUp)
    char *x16;      // 8-bit rows: packed rows of `dim` elements that hold their codes' values; else nullptr
    bool x8;        // kFfnGateUp: rows of 8-bit codes
    int act;
};

template <int DT> hipError_t launch_ffn(FfnKind kind, const FfnArgs &a, uint32_t num_cus, hipStream_t st);

}  // namespace hcclx
