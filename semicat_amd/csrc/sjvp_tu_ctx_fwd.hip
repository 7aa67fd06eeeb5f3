// Translation unit: forward kernels of the attention on keys of another length for one element type (SJVP_T).
#include <type_traits>

#include "sjvp_ctx_fwd.hpp"
#include "sjvp_ctx_launch.hpp"

namespace sjvp {

template <>
int ctx_forward<SJVP_T>(CtxParams p, const CtxPlan& plan, hipStream_t stream) {
    p.blocks = plan.blocks, p.splits = plan.splits;
    const int grid = (int)ctx_grid((int)plan.units, (int)plan.inner);
    return ctx_by_head(p.D, [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (!plan.few) return p.table ? launch(ctx_fwd<SJVP_T, HD, true>, grid, plan.smem, stream, p, kCtxThreads)
                                      : launch(ctx_fwd<SJVP_T, HD, false>, grid, plan.smem, stream, p, kCtxThreads);
        p.packed = plan.packed;
        const int rc = p.table ? launch(ctx_fwd_few<SJVP_T, HD, true>, grid, plan.smem, stream, p, kCtxThreads)
                               : launch(ctx_fwd_few<SJVP_T, HD, false>, grid, plan.smem, stream, p, kCtxThreads);
        if (rc != SJVP_OK || p.splits == 1) return rc;
        const int64_t threads = (int64_t)p.B * p.Hq * p.Lq * (HD / 8);
        return launch(ctx_join<SJVP_T, HD>, (int)((threads + kCtxThreads - 1) / kCtxThreads), 0, stream, p, kCtxThreads);
    });
}

}  // namespace sjvp
