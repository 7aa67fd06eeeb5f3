// Translation unit: forward kernels of the attention on keys of another length for one element type (SJVP_T).
#include <type_traits>

#include "sjvp_ctx_fwd.hpp"
#include "sjvp_ctx_launch.hpp"

namespace sjvp {

template <>
int ctx_forward<SJVP_T>(CtxParams p, const CtxPlan& plan, hipStream_t stream) {
    p.blocks = plan.blocks, p.splits = plan.splits;
    const int grid = (int)ctx_grid(plan.units, plan.inner);
    p.packed = plan.packed;
    return ctx_by_head(p.D, plan.dma, [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        const auto run = [&](auto bias, auto terms) {
            constexpr bool BIAS = decltype(bias)::value;
            constexpr int TERMS = decltype(terms)::value;
            if (!plan.few) return launch(ctx_fwd<SJVP_T, HD, BIAS, decltype(dma)::value, TERMS>, grid, plan.smem, stream, p, kCtxThreads);
            if constexpr (BIAS)
                if (plan.waves == 8) return launch(ctx_fwd_few<SJVP_T, HD, BIAS, TERMS, 8>, grid, plan.smem, stream, p, 512);
            return launch(ctx_fwd_few<SJVP_T, HD, BIAS, TERMS, 4>, grid, plan.smem, stream, p, 256);
        };
        const std::true_type yes;
        const std::false_type no;
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> two;
        const std::integral_constant<int, std::is_same_v<SJVP_T, Bf16> ? 3 : 2> most;
        const int rc = !p.rest.ptr ? p.table ? run(yes, one) : run(no, one)
                       : !p.table  ? run(no, two)
                                   : p.table_type == SJVP_FP32 ? run(yes, most) : run(yes, two);
        if (!plan.few) return rc;
        if (rc != SJVP_OK || p.splits == 1) return rc;
        int slices = 1;  // as in the kernel
        while (slices < p.splits && slices < 16) slices *= 2;
        const int64_t rows = (int64_t)p.B * p.Hq * p.Lq, per = 16 / slices;
        return launch(ctx_join<SJVP_T, HD>, (int)((rows + per - 1) / per), 0, stream, p, kCtxThreads);
    });
}

}  // namespace sjvp
