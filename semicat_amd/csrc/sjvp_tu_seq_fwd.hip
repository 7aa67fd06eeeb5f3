// Translation unit: forward kernels of the attention over packed sequences and over a paged cache for one element type (SJVP_T).
#include "sjvp_seq_fwd.hpp"
#include "sjvp_seq_launch.hpp"

namespace sjvp {

template <>
int seq_packed_fwd<SJVP_T>(SeqParams p, hipStream_t stream) {
    p.slots = (int)seq_slots(p, p.G, kCtxOwned), p.splits = 1, p.least = 0, p.most = INT_MAX;
    return seq_by_head(p.D, seq_dma(p, p.k, p.v), [&](auto hd, auto dma) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool DMA = decltype(dma)::value;
        return launch(seq_fwd<SJVP_T, HD, false, SeqFeed<HD, DMA>>, p.slots * p.Hkv, seq_tiles_bytes(HD), stream, p, kCtxThreads);
    });
}

template <>
int seq_paged<SJVP_T>(SeqParams p, bool e4m3, bool few, bool many, hipStream_t stream) {
    const int splits = p.splits;
    return seq_by_head(p.D, [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        int rc = SJVP_OK;
        if (few) {
            const auto run = [&](auto sets, auto bits8) {
                constexpr int NC = decltype(sets)::value;
                p.slots = (int)seq_slots(p, p.G, 16 * NC), p.least = 0, p.most = many ? kSeqFew : INT_MAX;
                const int smem = kCtxWaves * std::max(32 * (HD + 8) * 2, 16 * NC * (HD + 4 + 2) * 4);
                return launch(seq_few<SJVP_T, HD, decltype(bits8)::value, NC, kCtxWaves>, p.slots * p.Hkv * splits, smem, stream, p, kCtxThreads);
            };
            const std::integral_constant<int, 1> one;
            const std::integral_constant<int, 2> two;
            const std::true_type yes;
            const std::false_type no;
            rc = seq_sets(p) == 1 ? e4m3 ? run(one, yes) : run(one, no) : e4m3 ? run(two, yes) : run(two, no);
            if (rc != SJVP_OK) return rc;
        }
        if (many) {
            SeqParams m = p;
            m.slots = (int)seq_slots(p, p.G, kCtxOwned), m.least = few ? kSeqFew + 1 : 0, m.most = INT_MAX;
            rc = e4m3 ? launch(seq_fwd<SJVP_T, HD, true, PageFeed8<SJVP_T, HD>>, m.slots * p.Hkv, seq_tiles_bytes(HD), stream, m, kCtxThreads)
                      : launch(seq_fwd<SJVP_T, HD, true, PageFeed<HD>>, m.slots * p.Hkv, seq_tiles_bytes(HD), stream, m, kCtxThreads);
            if (rc != SJVP_OK) return rc;
        }
        if (!few || splits == 1) return rc;
        int slices = 1;  // as in the kernel
        while (slices < splits && slices < 16) slices *= 2;
        const int64_t rows = p.Hkv * (many ? (int64_t)(p.B + 2) * kSeqFew : (int64_t)p.T * p.G), per = 16 / slices;
        return launch(seq_join<SJVP_T, HD>, (int)((rows + per - 1) / per), 0, stream, p, kCtxThreads);
    });
}

}  // namespace sjvp
