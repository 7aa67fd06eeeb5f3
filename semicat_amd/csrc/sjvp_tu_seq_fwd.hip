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
int seq_paged<SJVP_T>(SeqParams p, const PagedPlan& plan, float* ws, bool e4m3, hipStream_t stream) {
    SeqParams m = p;
    const auto put = [&](SeqParams& x, const PagedPart& part, int least, int most) {
        x.least = least, x.most = most, x.splits = part.splits, x.split_tiles = part.split_tiles;
        x.stat = ws + part.stat, x.part = ws + part.part, x.used = reinterpret_cast<int*>(ws + part.used);
    };
    put(p, plan.few, 0, plan.has_many ? kSeqFew : INT_MAX);
    put(m, plan.many, plan.has_few ? kSeqFew + 1 : 0, INT_MAX);
    p.used_many = plan.has_many && plan.many.splits > 1 ? m.used : nullptr;
    return seq_by_head(p.D, [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        const auto few = [&](auto sets, auto bits8) {
            constexpr int NC = decltype(sets)::value;
            p.slots = (int)(plan.has_many ? (int64_t)(p.B + 2) * (kSeqFew / (16 * NC)) : seq_slots(p, p.G, 16 * NC));
            const auto run = [&](auto waves) {
                constexpr int WAVES = decltype(waves)::value;
                const int smem = WAVES * std::max(32 * (HD + 8) * 2, 16 * NC * (HD + 4 + 2) * 4);
                return launch(seq_few<SJVP_T, HD, decltype(bits8)::value, NC, WAVES>, p.slots * p.Hkv * p.splits, smem, stream, p, 64 * WAVES);
            };
            // Short caches: a workgroup of one wave, of which four times as many run at once (123 tokens on up to 43 each, 23 heads of 112: 12.6 us in place
            // of 20.9; 11 sequences of 71 tokens on 71, 32 heads of 128: 15.1 and 21.0); a few of them are faster with four waves (36 sequences
            // of 8 tokens on up to 65, 9 heads: 8.5 us and 11.1).
            const int64_t keys = p.pages.capacity;
            const bool alone = keys <= 64 || (keys <= 512 && 32 * (int64_t)p.slots * p.Hkv >= keys * compute_units());
            return alone ? run(std::integral_constant<int, 1>{}) : run(std::integral_constant<int, kCtxWaves>{});
        };
        const auto join = [&](const SeqParams& x) {
            if (x.splits == 1) return (int)SJVP_OK;
            int slices = 1;  // as in the kernel
            while (slices < x.splits && slices < 16) slices *= 2;
            const int64_t rows = x.Hkv * (x.most == kSeqFew ? (int64_t)(x.B + 2) * kSeqFew : (int64_t)x.T * x.G), per = 16 / slices;
            return launch(seq_join<SJVP_T, HD>, (int)((rows + per - 1) / per), 0, stream, x, kCtxThreads);
        };
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> two;
        const std::true_type yes;
        const std::false_type no;
        int rc = SJVP_OK;
        if (plan.has_few) {
            rc = seq_sets(p) == 1 ? e4m3 ? few(one, yes) : few(one, no) : e4m3 ? few(two, yes) : few(two, no);
            if (rc == SJVP_OK) rc = join(p);
        }
        if (rc != SJVP_OK || !plan.has_many) return rc;
        m.slots = (int)seq_slots(m, m.G, kCtxOwned);
        const int grid = m.slots * m.Hkv * m.splits;
        rc = e4m3 ? launch(seq_fwd<SJVP_T, HD, true, PageFeed8<SJVP_T, HD>>, grid, seq_tiles_bytes(HD), stream, m, kCtxThreads)
                  : launch(seq_fwd<SJVP_T, HD, true, PageFeed<HD>>, grid, seq_tiles_bytes(HD), stream, m, kCtxThreads);
        return rc == SJVP_OK ? join(m) : rc;
    });
}

}  // namespace sjvp
