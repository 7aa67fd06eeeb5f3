// How a call of the attention of sjvp_ctx.hpp is split over workgroups, and its launches, for the translation units.
#pragma once
#include "sjvp_ctx.hpp"
#include "sjvp_launch.hpp"

namespace sjvp {

// Head dimensions are padded to whole multiples of 32.
inline int ctx_padded(int D) { return (D + 31) / 32 * 32; }
inline int ctx_entries(const CtxParams& p) { return 2 * (p.far + kCtxPad) + 1; }
inline int ctx_tiles_bytes(int HD) { return 4 * kCtxTile * (HD + 8) * 2; }

// One launch's share of the work: `blocks` over the owned axis, `splits` of the looped one.
struct CtxPlan {
    bool few = false;      // forward: ctx_fwd_few
    int packed = 1;        // its heads to a block of rows,
    int waves = kCtxWaves;  // and waves to a workgroup
    int blocks = 1, splits = 1;
    int64_t units = 1, inner = 1;  // of ctx_work
    int smem = 0, skew = 0;
};

CtxPlan ctx_plan_fwd(const CtxParams& p);
CtxPlan ctx_plan_row(const CtxParams& p);
CtxPlan ctx_plan_col(const CtxParams& p);

template <typename T> int ctx_forward(CtxParams p, const CtxPlan& plan, hipStream_t stream);
// row: the row-owned launch (dQ, delta, bucket sums), else the column-owned one (dK, dV)
template <typename T> int ctx_backward(CtxParams p, const CtxPlan& plan, bool row, hipStream_t stream);

// Calls f with the padded head dimension as a constant.
template <typename F>
int ctx_by_head(int D, F&& f) {
    switch (ctx_padded(D)) {
        case 32: return f(std::integral_constant<int, 32>{});
        case 64: return f(std::integral_constant<int, 64>{});
        case 96: return f(std::integral_constant<int, 96>{});
        default: return f(std::integral_constant<int, 128>{});
    }
}

}  // namespace sjvp
