// Translation unit: backward kernels of the attention over packed sequences for one element type (SJVP_T).
#include "sjvp_seq_bwd.hpp"
#include "sjvp_seq_launch.hpp"

namespace sjvp {

template <>
int seq_packed_bwd<SJVP_T>(SeqParams p, hipStream_t stream) {
    const bool row_dma = seq_dma(p, p.k, p.v), col_dma = seq_dma(p, p.q, p.g) && row_dma;  // (at D = 128 the column-owned one has K and V in LDS too)
    const int splits = p.splits;
    p.slots = (int)seq_slots(p, p.G, kCtxOwned);
    int rc = seq_by_head(p.D, row_dma, [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool DMA = decltype(dma)::value;
        return launch(seq_bwd_row<SJVP_T, HD, DMA>, p.slots * p.Hkv, seq_tiles_bytes(HD), stream, p, kCtxThreads);
    });
    if (rc != SJVP_OK || !p.dk.ptr) return rc;
    p.slots = (int)seq_slots(p, 1, kCtxOwned);
    p.splits = splits;
    return seq_by_head(p.D, col_dma, [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool DMA = decltype(dma)::value;
        const int grid = p.slots * p.Hkv * p.splits;
        int rc;
        if constexpr (HD > 64) rc = launch(seq_bwd_col_pair<SJVP_T, HD, DMA>, grid, 2 * seq_tiles_bytes(HD) + 4 * kCtxStats, stream, p, 2 * kCtxThreads);
        else rc = launch(seq_bwd_col<SJVP_T, HD, DMA>, grid, seq_tiles_bytes(HD) + 4 * kCtxStats, stream, p, kCtxThreads);
        if (rc != SJVP_OK || p.splits == 1) return rc;
        return launch(seq_sum<SJVP_T, HD>, (int)((2 * (int64_t)p.Hkv * p.T * (HD / 8) + kCtxThreads - 1) / kCtxThreads), 0, stream, p, kCtxThreads);
    });
}

}  // namespace sjvp
