// Translation unit: backward kernels of the attention on keys of another length for one element type (SJVP_T).
#include <type_traits>

#include "sjvp_ctx_bwd.hpp"
#include "sjvp_ctx_launch.hpp"

namespace sjvp {

template <>
int ctx_backward<SJVP_T>(CtxParams p, const CtxPlan& plan, bool row, hipStream_t stream) {
    p.blocks = plan.blocks, p.splits = plan.splits, p.cols = !row;
    const int grid = (int)ctx_grid(plan.units, plan.inner);
    return ctx_by_head(p.D, plan.dma, [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool DMA = decltype(dma)::value;
        int rc;
        if (row) rc = p.table ? launch(ctx_bwd_row<SJVP_T, HD, true, DMA>, grid, plan.smem, stream, p, kCtxThreads)
                              : launch(ctx_bwd_row<SJVP_T, HD, false, DMA>, grid, plan.smem, stream, p, kCtxThreads);
        else rc = p.table ? launch(ctx_bwd_col<SJVP_T, HD, true, DMA>, grid, plan.smem, stream, p, kCtxThreads)
                          : launch(ctx_bwd_col<SJVP_T, HD, false, DMA>, grid, plan.smem, stream, p, kCtxThreads);
        if (rc != SJVP_OK || p.splits == 1) return rc;
        const int64_t rows = row ? (int64_t)p.B * p.Hq * p.Lq : 2 * (int64_t)p.B * p.Hkv * p.Lk;
        return launch(ctx_sum<SJVP_T, HD>, (int)((rows * (HD / 8) + kCtxThreads - 1) / kCtxThreads), 0, stream, p, kCtxThreads);
    });
}

template <>
int ctx_backward_one<SJVP_T>(CtxParams p, const CtxPlan& plan, hipStream_t stream) {
    p.blocks = p.splits = 1, p.packed = plan.packed;
    const int grid = (int)ctx_grid(plan.units, 1);
    const auto run = [&](auto bias, auto dma) {
        constexpr bool BIAS = decltype(bias)::value, DMA = decltype(dma)::value;
        return plan.waves == 8 ? launch(ctx_bwd_one<SJVP_T, BIAS, DMA, 8>, grid, plan.smem, stream, p, 512)
                               : launch(ctx_bwd_one<SJVP_T, BIAS, DMA, 4>, grid, plan.smem, stream, p, 256);
    };
    const std::true_type yes;
    const std::false_type no;
    return p.table ? plan.dma ? run(yes, yes) : run(yes, no) : plan.dma ? run(no, yes) : run(no, no);
}

}  // namespace sjvp
