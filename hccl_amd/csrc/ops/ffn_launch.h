// Which kernel computes a product: instantiated per type in ffn_bf16.hip and ffn_f16.hip.
#pragma once
#include "ops/ffn_gemm.h"
#include "ops/ffn_thin.h"

namespace hcclx {

// Rows per rank, if all have as many, up to which the forward products read the weights straight into registers.
constexpr uint32_t kThinRows = 32;
inline bool thin(const FfnRows &s) { return s.most <= static_cast<uint64_t>(s.n) * kThinRows; }

// Rows per rank up to which products take tiles of half a whole tile's height and width.
constexpr uint32_t kSmallRows = 128;
inline bool small_tiles(const FfnRows &s) { return s.most <= static_cast<uint64_t>(s.n) * kSmallRows; }

template <int DT, int KIND>
hipError_t launch_forward(const FfnArgs &a, uint32_t num_cus, hipStream_t st)
{
    const FfnRows &s = a.rows;
    if (s.most == 0) return hipSuccess;
    if (!thin(s)) return ffn::run<DT, KIND>(a, small_tiles(s), num_cus, st);
    const bool x8 = a.x8;
    if (s.most <= static_cast<uint64_t>(s.n) * 16) {
        ffn::launch_thin<DT, KIND, 1>(a, x8, st);
    } else {
        ffn::launch_thin<DT, KIND, 2>(a, x8, st);
    }
    return hipGetLastError();
}

template <int DT>
hipError_t launch_ffn_widen(const FfnArgs &a, hipStream_t st)
{
    if (a.rows.most == 0 || thin(a.rows)) return hipSuccess;   // the thin kernel reads the codes
    HCCLX_LAUNCH((ffn::k_ffn_widen<DT>), dim3((a.rows.most + 3) / 4), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_ffn(FfnKind kind, const FfnArgs &a, uint32_t num_cus, hipStream_t st)
{
    switch (kind) {
        case kFfnGateUp: return launch_forward<DT, kFfnGateUp>(a, num_cus, st);
        case kFfnDown: return launch_forward<DT, kFfnDown>(a, num_cus, st);
        case kFfnGradHidden: return ffn::run<DT, kFfnGradHidden>(a, small_tiles(a.rows), num_cus, st);
        case kFfnGradInput: return ffn::run<DT, kFfnGradInput>(a, small_tiles(a.rows), num_cus, st);
        default: return ffn::run<DT, kFfnGradWeights>(a, small_tiles(a.rows), num_cus, st);
    }
}

}  // namespace hcclx
