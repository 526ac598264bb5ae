// Which kernel computes a product: instantiated per type in ffn_bf16.hip and ffn_f16.hip.  A choice goes by the sizes and by the
// bound on the rows of all ranks, from which the rows of a rank are taken as if all had as many; whatever they turn out to be on
// the device, every kernel is right for them.  (A plan whose bound is far above what a launch then has runs the kernels of the bound.)
#pragma once
#include "ops/ffn_gemm.h"
#include "ops/ffn_thin.h"

namespace hcclx {
namespace ffn {

// Products with few rows read the weights; what counts is how many bytes are on their way.  Tiles of 128 x 128 keep 48 KiB of
// weights per CU on their way and read the rows' operand once per tile, but have to be as many as the CUs; the thin kernel
// has eight wavefronts per 16 columns and reads the rows' operand that often.  Both products, weights from memory, thin : tiles, us:
// up to a quarter of a round of tiles, 2 ranks x 4096 x 2048 (64 tiles of the first product), 1 row 26.5 : 60, 64 rows 55 : 64; 1 rank
// (32), 64 rows 42 : 62; 1 x 7168 x 2048, 64 rows 74 : 88.  Up to a round, 4 ranks x 7168 x 2048 (128 tiles), 1 row 75 : 95, 8 rows
// 82 : 96, 64 rows 182 : 106; 8 x 4096 x 1024 (128), 8 rows 52 : 60, 64 rows 115 : 64.  A full round, 8 x 7168 x 2048 (256), 1 row
// 138 : 146, 4 rows 144 : 138, 16 rows 174 : 139; 16 x 2048 x 1024 (256), 1 row 50 : 56, 8 rows 55 : 56, 16 rows 60 : 57.  What the rule
// leaves: a single row at a full round, and 9 to 16 rows at half of one (4 x 16 x 7168 x 2048 92 : 97, 8 x 16 x 4096 x 1024 58 : 60.5).
template <int KIND>
bool thin(const FfnRows &s, uint32_t cus)
{
    const uint64_t tiles = static_cast<uint64_t>(s.n) * ((columns<KIND>(s) + kTileCols<KIND> / 2 - 1) / (kTileCols<KIND> / 2));
    const uint64_t rows = (s.most + s.n - 1) / s.n;
    return (rows <= 64 && tiles <= cus / 4) || (rows <= 8 && tiles < cus);
}

// Workgroups of eight columns instead of sixteen, while no CU gets two of them.  The block, 1 row, halves : sixteens, us: 1 rank
// 4096 x 512 14.5 : 15.6, 4096 x 2048 (128 workgroups of sixteen) 16.2 : 17.3, 16 rows 18.9 : 20.3; 2 ranks (256) 31 : 25.
inline bool halves(const FfnRows &s, uint32_t cus) { return static_cast<uint64_t>(s.n) * ((s.hidden + 15) / 16) <= cus / 2; }

// Rows of a rank up to which tiles of 128 x 128 are taken: a whole tile would be half empty.  8 ranks x 4096 x 2048, small : whole
// tiles, us: 64 rows, forward 99 : 121, gradients of the rows 134 : 144; 128 rows 115 : 125, 140 : 152; 160 rows, forward 146 : 124.
constexpr uint32_t kSmallRows = 128;

// Of those, which: a round of tiles of 128 x 256 takes 1.3 times as long as one of 128 x 128, and there are as many rounds as the
// fullest CU has tiles.  Block of 8 ranks, 64 rows, wide in both products : small, us: 7168 x 2112 (132 tiles in a round : 264 in
// two) 174 : 195, 6144 x 2560 180 : 200; 7168 x 2048 (256 in a round) 180 : 152, 4096 x 1024 91 : 64.
template <int KIND>
Cut cut_of(const FfnRows &s, uint32_t cus)
{
    if (s.most > static_cast<uint64_t>(s.n) * kSmallRows) return kCutWhole;
    auto rounds = [&](uint32_t cols) {
        const uint64_t tiles = static_cast<uint64_t>(s.n) * ((columns<KIND>(s) + cols - 1) / cols);
        return (tiles + cus - 1) / cus;
    };
    return 13 * rounds(kTileCols<KIND>) < 10 * rounds(kTileCols<KIND> / 2) ? kCutWide : kCutSmall;
}

template <int DT, int KIND>
hipError_t launch(const FfnArgs &a, uint32_t cus, hipStream_t st)
{
    const FfnRows &s = a.rows;
    if constexpr (KIND == kFfnGateUp || KIND == kFfnDown) {
        if (s.most != 0 && thin<KIND>(s, cus)) {
            const uint64_t rows = (s.most + s.n - 1) / s.n;
            if (rows <= 16) {
                if (KIND == kFfnGateUp && halves(s, cus)) {
                    launch_thin<DT, KIND, 1, KIND == kFfnGateUp>(a, st);
                } else {
                    launch_thin<DT, KIND, 1, false>(a, st);
                }
            } else if (rows <= 32) {
                launch_thin<DT, KIND, 2, false>(a, st);
            } else {
                launch_thin<DT, KIND, 4, false>(a, st);
            }
            return hipGetLastError();
        }
        if (KIND == kFfnGateUp && a.x8 && s.most != 0) {   // (the thin kernel reads the codes)
            HCCLX_LAUNCH((k_ffn_widen<DT>), dim3(s.most), dim3(256), 0, st, a);
        }
    }
    return run<DT, KIND>(a, cut_of<KIND>(s, cus), cus, st);
}

}  // namespace ffn

template <int DT>
hipError_t launch_ffn(FfnKind kind, const FfnArgs &a, uint32_t num_cus, hipStream_t st)
{
    switch (kind) {
        case kFfnGateUp: return ffn::launch<DT, kFfnGateUp>(a, num_cus, st);
        case kFfnDown: return ffn::launch<DT, kFfnDown>(a, num_cus, st);
        case kFfnGradHidden: return ffn::launch<DT, kFfnGradHidden>(a, num_cus, st);
        case kFfnGradInput: return ffn::launch<DT, kFfnGradInput>(a, num_cus, st);
        default: return ffn::launch<DT, kFfnGradWeights>(a, num_cus, st);
    }
}

}  // namespace hcclx
