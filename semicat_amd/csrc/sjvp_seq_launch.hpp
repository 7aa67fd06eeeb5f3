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

// Sets of 16 rows to a block of seq_few.
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
// e4m3: pages of 8-bit numbers; few, many: which of the two kernels serve the call
template <typename T> int seq_paged(SeqParams p, bool e4m3, bool few, bool many, hipStream_t stream);
int paged_copy(const SeqParams& p, bool e4m3, bool fp16, bool write, hipStream_t stream);

}  // namespace sjvp
