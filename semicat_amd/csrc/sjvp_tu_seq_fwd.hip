// Translation unit: forward kernels of the attention over packed sequences and over a paged cache for one element type (SJVP_T).
#include "sjvp_seq_fwd.hpp"
#include "sjvp_seq_launch.hpp"

namespace sjvp {

template <>
int seq_packed_fwd<SJVP_T>(SeqParams p, hipStream_t stream) {
    p.slots = (int)seq_slots(p, p.G, kCtxOwned), p.splits = 1, p.least = 0, p.most = INT_MAX;
    return ctx_by_head(p.D, seq_dma(p, p.k, p.v), [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool DMA = decltype(dma)::value;
        return launch(seq_fwd<SJVP_T, HD, false, SeqFeed<HD, DMA>>, p.slots * p.Hkv, ctx_tiles_bytes(HD, DMA), stream, p, kCtxThreads);
    });
}

template <>
int seq_paged<SJVP_T>(SeqParams p, bool e4m3, bool few, bool many, hipStream_t stream) {
    const int splits = p.splits;
    const auto with = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool DMA = HD != 96;  // (twelve pieces to a row do not fit the permutation of LDS-DMA tiles)
        int rc = SJVP_OK;
        if (few) {
            p.slots = (int)seq_slots(p, p.G, 32), p.least = 0, p.most = many ? kSeqFew : INT_MAX;
            const int grid = p.slots * p.Hkv * splits, smem = kCtxWaves * 32 * (HD + 4 + 2) * 4;
            rc = e4m3 ? launch(seq_few<SJVP_T, HD, true, kCtxWaves>, grid, smem, stream, p, kCtxThreads)
                      : launch(seq_few<SJVP_T, HD, false, kCtxWaves>, grid, smem, stream, p, kCtxThreads);
            if (rc != SJVP_OK) return rc;
        }
        if (many) {
            SeqParams m = p;
            m.slots = (int)seq_slots(p, p.G, kCtxOwned), m.least = few ? kSeqFew + 1 : 0, m.most = INT_MAX;
            rc = e4m3 ? launch(seq_fwd<SJVP_T, HD, true, PageFeed8<SJVP_T, HD>>, m.slots * p.Hkv, ctx_tiles_bytes(HD, false), stream, m, kCtxThreads)
                      : launch(seq_fwd<SJVP_T, HD, true, PageFeed<HD, DMA>>, m.slots * p.Hkv, ctx_tiles_bytes(HD, DMA), stream, m, kCtxThreads);
            if (rc != SJVP_OK) return rc;
        }
        if (!few || splits == 1) return rc;
        int slices = 1;  // as in the kernel
        while (slices < splits && slices < 16) slices *= 2;
        const int64_t rows = p.Hkv * (many ? (int64_t)(p.B + 2) * kSeqFew : (int64_t)p.T * p.G), per = 16 / slices;
        return launch(seq_join<SJVP_T, HD>, (int)((rows + per - 1) / per), 0, stream, p, kCtxThreads);
    };
    switch (ctx_padded(p.D)) {
        case 32: return with(std::integral_constant<int, 32>{});
        case 64: return with(std::integral_constant<int, 64>{});
        case 96: return with(std::integral_constant<int, 96>{});
        default: return with(std::integral_constant<int, 128>{});
    }
}

}  // namespace sjvp
