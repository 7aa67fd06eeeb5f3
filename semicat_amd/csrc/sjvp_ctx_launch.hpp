// How a call of the attention of sjvp_ctx.hpp is split over workgroups, and its launches, for the translation units.
#pragma once
#include "sjvp_ctx.hpp"
#include "sjvp_launch.hpp"

namespace sjvp {

// Head dimensions are padded to whole multiples of 32.
inline int ctx_padded(int D) { return (D + 31) / 32 * 32; }
inline int ctx_entries(const CtxParams& p) { return 2 * (p.far + kCtxPad) + 1; }
inline int ctx_tiles_bytes(int HD, bool dma) { return 4 * kCtxTile * (HD + (dma ? 0 : 8)) * 2; }

// Rows that LDS-DMA copies take: 16-byte aligned, of whole 16-byte pieces.  (At head dimensions 65 to 96 a row has twelve pieces, which the
// permutation of the pieces in LDS does not fit.)
inline bool ctx_aligned(const CtxView& v) {
    return (reinterpret_cast<uintptr_t>(v.ptr) & 15) == 0 && ((v.sb | v.sh | v.sl) & 7) == 0;
}
inline bool ctx_dma(const CtxParams& p, const CtxView& a, const CtxView& b) {
    return p.D % 8 == 0 && ctx_padded(p.D) != 96 && ctx_aligned(a) && ctx_aligned(b);
}

// One launch's share of the work: `blocks` over the owned axis, `splits` of the looped one.
struct CtxPlan {
    bool few = false;      // forward: ctx_fwd_few
    int packed = 1;        // its heads to a block of rows (ctx_bwd_one: sets of dS tiles),
    int waves = kCtxWaves;  // and waves to a workgroup
    int blocks = 1, splits = 1;
    int64_t units = 1, inner = 1;  // of ctx_work
    int smem = 0;
    bool dma = false;              // tiles by LDS-DMA
};

CtxPlan ctx_plan_fwd(const CtxParams& p);
CtxPlan ctx_plan_row(const CtxParams& p);
CtxPlan ctx_plan_col(const CtxParams& p);
bool ctx_plan_one(const CtxParams& p, CtxPlan& plan);  // whether one launch does the backward

template <typename T> int ctx_forward(CtxParams p, const CtxPlan& plan, hipStream_t stream);
// row: the row-owned launch (dQ, delta, bucket sums), else the column-owned one (dK, dV)
template <typename T> int ctx_backward(CtxParams p, const CtxPlan& plan, bool row, hipStream_t stream);

template <typename T> int ctx_backward_one(CtxParams p, const CtxPlan& plan, hipStream_t stream);

// Calls f with the padded head dimension, and whether tiles come by LDS-DMA, as constants.
template <typename F>
int ctx_by_head(int D, bool dma, F&& f) {
    const auto with = [&](auto hd) { return dma ? f(hd, std::true_type{}) : f(hd, std::false_type{}); };
    switch (ctx_padded(D)) {
        case 32: return with(std::integral_constant<int, 32>{});
        case 64: return with(std::integral_constant<int, 64>{});
        case 96: return f(std::integral_constant<int, 96>{}, std::false_type{});
        default: return with(std::integral_constant<int, 128>{});
    }
}

}  // namespace sjvp
