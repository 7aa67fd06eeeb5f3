// Launches of the attention over packed sequences and over a paged cache, for the translation units.
#pragma once
#include <algorithm>
#include <climits>
#include <type_traits>
#include "sjvp_ctx_launch.hpp"
#include "sjvp_seq.hpp"

namespace sjvp {

// Blocks of R rows that the segments of a call can have (see seq_block).
inline int64_t seq_slots(const SeqParams& p, int heads, int R) { return (int64_t)p.T * heads / R + p.B + 2; }

// Sets of 16 rows to a block of seq_few: one where a sequence has up to 16 rows on average, which leaves registers for four waves to a SIMD (a token each of
// 64 sequences on 1200 to 4096, Hq=16 Hkv=4 D=128 e4m3: 41.5 us, two sets 48.2; six tokens of 16, 24 rows: 25.9 and 22.3).
inline int seq_sets(const SeqParams& p) { return (int64_t)p.T * p.G <= 16 * (int64_t)p.B ? 1 : 2; }

inline bool seq_dma(const SeqParams& p, const CtxView& a, const CtxView& b) { return p.D % 8 == 0 && ctx_aligned(a) && ctx_aligned(b); }
inline int seq_tiles_bytes(int HD) { return 4 * kCtxTile * (HD == 96 ? 128 : HD) * 2; }

// Calls f with the padded head dimension, and, where it is wanted, whether tiles come by LDS-DMA, as constants.
template <typename F>
int seq_by_head(int D, F&& f) {
    switch (ctx_padded(D)) {
        case 32: return f(std::integral_constant<int, 32>{});
        case 64: return f(std::integral_constant<int, 64>{});
        case 96: return f(std::integral_constant<int, 96>{});
        default: return f(std::integral_constant<int, 128>{});
    }
}
template <typename F>
int seq_by_head(int D, bool dma, F&& f) {
    return seq_by_head(D, [&](auto hd) { return dma ? f(hd, std::true_type{}) : f(hd, std::false_type{}); });
}

template <typename T> int seq_packed_fwd(SeqParams p, hipStream_t stream);
template <typename T> int seq_packed_bwd(SeqParams p, hipStream_t stream);
// How a call of the paged attention is served: by seq_few, which splits long sequences over workgroups and takes any number of rows, or, where
// the sequences have 128 rows on average and blocks of 128 rows fill half of the compute units (an eighth with tables of 1024 positions or more), the longer
// sequences by seq_fwd (paged_plan).  Scratch of each: places in floats.
struct PagedPart {
    int splits = 1, split_tiles = 1;
    size_t stat = 0, part = 0, used = 0;
};
struct PagedPlan {
    bool has_few = true, has_many = false;
    PagedPart few, many;
    size_t total = 0;
};
// e4m3: pages of 8-bit numbers
template <typename T> int seq_paged(SeqParams p, const PagedPlan& plan, float* ws, bool e4m3, hipStream_t stream);
int paged_copy(const SeqParams& p, bool e4m3, bool fp16, bool write, hipStream_t stream);

}  // namespace sjvp
