// Translation unit: forward kernels of the attention on keys of another length for one element type (SJVP_T).
#include <type_traits>

#include "sjvp_ctx_fwd.hpp"
#include "sjvp_ctx_launch.hpp"

namespace sjvp {

template <>
int ctx_forward<SJVP_T>(CtxParams p, const CtxPlan& plan, hipStream_t stream) {
    p.blocks = plan.blocks, p.splits = plan.splits;
    const int grid = (int)ctx_grid((int)plan.units, (int)plan.inner);
    return ctx_by_head(p.D, plan.dma, [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool DMA = decltype(dma)::value;
        if (!plan.few) return p.table ? launch(ctx_fwd<SJVP_T, HD, true, DMA>, grid, plan.smem, stream, p, kCtxThreads)
                                      : launch(ctx_fwd<SJVP_T, HD, false, DMA>, grid, plan.smem, stream, p, kCtxThreads);
        p.packed = plan.packed;
        const auto few = [&](auto waves) {
            constexpr int W = decltype(waves)::value;
            return p.table ? launch(ctx_fwd_few<SJVP_T, HD, true, W>, grid, plan.smem, stream, p, 64 * W)
                           : launch(ctx_fwd_few<SJVP_T, HD, false, W>, grid, plan.smem, stream, p, 64 * W);
        };
        const int rc = plan.waves == 8 ? few(std::integral_constant<int, 8>{}) : few(std::integral_constant<int, 4>{});
        if (rc != SJVP_OK || p.splits == 1) return rc;
        int slices = 1;  // as in the kernel
        while (slices < p.splits && slices < 16) slices *= 2;
        const int64_t rows = (int64_t)p.B * p.Hq * p.Lq, per = 16 / slices;
        return launch(ctx_join<SJVP_T, HD>, (int)((rows + per - 1) / per), 0, stream, p, kCtxThreads);
    });
}

}  // namespace sjvp
