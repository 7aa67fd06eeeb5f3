// Translation unit: forward kernels of the attention on keys of another length for one element type (SJVP_T).
#include <type_traits>

#include "sjvp_ctx_fwd.hpp"
#include "sjvp_ctx_launch.hpp"

namespace sjvp {

template <>
int ctx_forward<SJVP_T>(CtxParams p, const CtxPlan& plan, hipStream_t stream) {
    p.blocks = plan.blocks, p.splits = plan.splits;
    const int grid = (int)ctx_grid((int)plan.units, (int)plan.inner);
    p.packed = plan.packed;
    return ctx_by_head(p.D, plan.dma, [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        const auto run = [&](auto bias, auto rest) {
            constexpr bool BIAS = decltype(bias)::value, REST = decltype(rest)::value;
            if (!plan.few) return launch(ctx_fwd<SJVP_T, HD, BIAS, decltype(dma)::value, REST>, grid, plan.smem, stream, p, kCtxThreads);
            return plan.waves == 8 ? launch(ctx_fwd_few<SJVP_T, HD, BIAS, REST, 8>, grid, plan.smem, stream, p, 512)
                                   : launch(ctx_fwd_few<SJVP_T, HD, BIAS, REST, 4>, grid, plan.smem, stream, p, 256);
        };
        const std::true_type yes;
        const std::false_type no;
        const int rc = p.table ? p.rest.ptr ? run(yes, yes) : run(yes, no) : p.rest.ptr ? run(no, yes) : run(no, no);
        if (!plan.few) return rc;
        if (rc != SJVP_OK || p.splits == 1) return rc;
        int slices = 1;  // as in the kernel
        while (slices < p.splits && slices < 16) slices *= 2;
        const int64_t rows = (int64_t)p.B * p.Hq * p.Lq, per = 16 / slices;
        return launch(ctx_join<SJVP_T, HD>, (int)((rows + per - 1) / per), 0, stream, p, kCtxThreads);
    });
}

}  // namespace sjvp
