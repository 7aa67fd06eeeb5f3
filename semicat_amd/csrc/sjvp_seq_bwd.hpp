// Backward kernels of the attention over packed sequences (sjvp_seq.hpp).
//
//   dP = dO V^T,  delta = rowsum(dO * O),  dS = P (dP - delta)
//   dQ = scale dS K,  dK = scale sum_heads dS^T Q,  dV = sum_heads P^T dO
//
// A row-owned launch (dQ, delta) and a column-owned one (dK, dV), both of which recompute P: 3 + 4 contractions against the 5 of a
// single launch, whose dQ would be summed over workgroups by atomics in an order that changes from run to run.
#pragma once
#include "sjvp_seq_fwd.hpp"

namespace sjvp {

// 32 rows' numbers in LDS as the registers of a score tile
__device__ __forceinline__ f32x16 seq_of_rows(const float* rows, int h) {
    f32x16 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 four = *reinterpret_cast<const f32x4*>(rows + 8 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = four[j];
    }
    return x;
}

// Whether one of a wave's scores is not finite.
__device__ __forceinline__ bool some_not_finite(const f32x16& a, const f32x16& b) {
    float zero = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) zero = __builtin_fmaf(a[r], 0.0f, __builtin_fmaf(b[r], 0.0f, zero));
    return __builtin_amdgcn_ballot_w64(zero != 0.0f) != 0;
}

// Whether some wave says so, in the x-th tile, behind whose contractions is a barrier.  (One that leaves copies to LDS in flight, unlike a barrier
// with a reduction.)
__device__ __forceinline__ bool some_wave(int* last, int x, bool some, int lane) {
    if (some && lane == 0) *last = x + 1;
    workgroup_barrier();
    return __builtin_amdgcn_readfirstlane(*last) == x + 1;
}

// Row-owned: four waves of 32 query rows (of the heads that share a key head) share tiles of 64 keys.  Four sequences of 1500 to 6000 tokens, Hq=16 Hkv=4
// D=128, causal: 392 us = 1.06 PFLOP/s, the matrix unit busy 59 %; its waits are those between the two contractions of a tile, with two waves to a SIMD
// for registers.
template <typename T, int HD, bool DMA>
__global__ __launch_bounds__(kCtxThreads, HD <= 64 ? 3 : 2) void seq_bwd_row(SeqParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = SeqTile<HD>::kElems;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);  // K [2], V [2]
    __shared__ int hurt;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % p.Hkv;
    const SeqBlock b = seq_block_long_first<kCtxOwned>(p, blockIdx.x / p.Hkv, p.G, false, lane);
    if (!b.some) return;
    const int all = b.tokens * p.G;
    const SeqKeys<false> keys(p, b);
    const int r0 = b.row0 + 32 * wave, rows = min(max(all - r0, 0), 32);
    const SeqRow mine(p, hk, min(r0 + (lane & 31), all - 1));
    const bool ok = (lane & 31) < rows;
    const int limit = keys.seen(p, mine.token);
    const int n = keys.seen(p, (min(b.row0 + kCtxOwned, all) - 1) / p.G), whole = keys.seen(p, b.row0 / p.G);
    const int n_wave = rows > 0 ? keys.seen(p, (r0 + rows - 1) / p.G) : 0;
    const int nt = (n + kCtxTile - 1) / kCtxTile;
    SeqFeed<HD, DMA> feed(p, b, hk, tid);
    SeqTile<HD> at(tiles, lane);
    constexpr int kHalf = 32 * SeqTile<HD>::kLd * 2, kBytes = SeqTile<HD>::kBytes;
    const auto k_place = [&](int t) { return tiles + (t & 1) * kTile; };
    const auto v_place = [&](int t) { return tiles + (2 + (t & 1)) * kTile; };
    if (nt) feed.request(p, 0, n, k_place(0), v_place(0), wave);
    if (tid == 0) hurt = 0;

    const int64_t token = b.token + mine.token, stat = (int64_t)mine.hq * p.T + token;
    const f32x2 ml = ok && limit > 0 ? *reinterpret_cast<const f32x2*>(p.lse + 2 * stat) : f32x2{0.0f, 0.0f};
    const bool some = ml[1] != 0.0f;         // a row that sees no key has no gradient, whatever its cotangent,
    const bool scored = some && limit != 1;  // one that sees one key none of its score: exactly none, not what rounding leaves
    u32x4 own_q[HD / 16], own_g[HD / 16];
    own_operands<HD>(own_q, p.q.head(0, mine.hq) + token * p.q.sl, ok, h, p.D);
    own_operands<HD>(own_g, p.g.head(0, mine.hq) + token * p.g.sl, some, h, p.D);
    const f32x2 less_factor = row_stat(ml);
    const float less = less_factor[0], factor = less_factor[1];
    if (nt) feed.deliver(p, k_place(0), v_place(0), tid);
    // delta, from o where a row sees many keys.  Few keys leave more of o's rounding in it than the gradients are rounded by (causal L=64 D=64: dq
    // 1.60 times as far off in norm as rounding it alone, 1.42 with the delta of unrounded numbers), so blocks of up to two tiles, which LDS
    // holds at once, form it as the sum of P dP.
    float delta = 0.0f;
    const bool at_once = nt <= 2;
    if (at_once) {
        if (nt == 2) {
            feed.request(p, 1, n, k_place(1), v_place(1), wave);
            feed.deliver(p, k_place(1), v_place(1), tid);
        }
        feed.arrived();
        workgroup_barrier();
        for (int u = 0; u < 2 * nt; ++u) {
            if (32 * u >= n_wave) break;
            const f32x16 s = at.template scores<T>(u * kHalf, own_q), dp = at.template scores<T>(2 * kBytes + u * kHalf, own_g);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (32 * u + tile_row(r, 0) < limit - 4 * h) delta = __builtin_fmaf(fast_exp2(__builtin_fmaf(s[r], p.c, -less)), dp[r], delta);
        }
        delta = factor == 0.0f ? 0.0f : halves_sum(delta) * factor;
    } else {
        const elem_t* o = p.o.head(0, mine.hq) + token * p.o.sl;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
            const u32x4 x = some ? load_chunk(o, 16 * c + 8 * h, p.D) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 32; e += 16) delta += T::to_float((elem_t)(own_g[c][j] >> e)) * T::to_float((elem_t)(x[j] >> e));
        }
        delta = halves_sum(delta);
        feed.arrived();
        workgroup_barrier();
    }
    if (h == 0 && ok) {
        const int64_t every = (int64_t)p.Hq * p.T;
        const f32x2 folded = row_stat_folded(ml);
        p.folded[stat] = folded[0], p.folded[every + stat] = folded[1], p.folded[2 * every + stat] = -delta;
    }
    const float less_delta = -delta * factor;  // P (dP - delta) = exponential * (factor dP + less_delta)
    f32x16 acc[HD / 32] = {};
    int step = kBytes;
    const auto tile = [&](int t, auto masked) {
        const int key = t * kCtxTile;
        const bool more = t + 1 < nt && !at_once;  // (both tiles of a short block are there, and other waves may still read the second one for delta)
        if (more) feed.request(p, t + 1, n, k_place(t + 1), v_place(t + 1), wave);
        f32x16 s[2], ds[2];
        s[0] = s[1] = ds[0] = ds[1] = f32x16{};
        bool some = false;
        if (key < n_wave) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    s[u] = Mma32<T>::run(at.rows(u * kHalf, c), own_q[c], s[u]);
                    ds[u] = Mma32<T>::run(at.rows(2 * kBytes + u * kHalf, c), own_g[c], ds[u]);
                }
            reads_ahead<HD / 8, 2, 2, 2>();
            if constexpr (decltype(masked)::value) some = some_not_finite(s[0], s[1]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    ds[u][r] = fast_exp2(__builtin_fmaf(s[u][r], p.c, -less)) * __builtin_fmaf(ds[u][r], factor, less_delta);
                    if constexpr (decltype(masked)::value)
                        if (32 * u + tile_row(r, 0) >= limit - key - 4 * h) ds[u][r] = 0.0f;
                }
                if constexpr (!decltype(masked)::value) at.template add_columns<T>(acc, u * kHalf, ds[u]);
            }
        }
        if constexpr (decltype(masked)::value) {
            // (a hidden row of V has ended in a zero of dS, one of K would meet that zero in the contraction)
            if (p.causal && some_wave(&hurt, t, some, lane)) {
                add_not_finite<T, HD>(acc, k_place(t), 0, min(limit - key, kCtxTile), 0.0f, h);
                workgroup_barrier();
                keep_finite<T, HD, kCtxThreads>(k_place(t), tid);
                workgroup_barrier();
            }
            if (key < n_wave)
#pragma unroll
                for (int u = 0; u < 2; ++u) at.template add_columns<T>(acc, u * kHalf, ds[u]);
        }
        at.move(step);
        step = -step;
        if (more) feed.deliver(p, k_place(t + 1), v_place(t + 1), tid);
        feed.arrived();
        workgroup_barrier();
    };
    const int free = min(whole / kCtxTile, nt);
    int t = 0;
    for (; t < free; ++t) tile(t, std::false_type{});
    for (; t < nt; ++t) tile(t, std::true_type{});
    store_rows_at<T, HD>(acc, scored ? p.scale : 0.0f, rows, tiles + wave * 32 * (HD + 8), lane, p.D, [&](int row) {
        const SeqRow to(p, hk, r0 + row);
        return p.dq.head(0, to.hq) + (int64_t)(b.token + to.token) * p.dq.sl;
    });
}

// What the column-owned launches have in common: the block of keys, the heads of a split, and the tiles of 64 query rows that see a key of the block,
// head by head.
struct SeqCols {
    int hk, split, ta, tb, first_head, heads, tiles;
    SeqBlock b;
    __device__ __forceinline__ SeqCols(const SeqParams& p, int lane)
        : hk(blockIdx.x % p.Hkv), split(blockIdx.x / p.Hkv % p.splits),  // (splits side by side: they are equally long)
          b(seq_block_long_first<kCtxOwned>(p, blockIdx.x / p.Hkv / p.splits, 1, true, lane)) {
        const int keys = SeqKeys<false>(p, b).keys;
        ta = p.causal ? b.row0 / kCtxTile : 0, tb = (keys + kCtxTile - 1) / kCtxTile;
        first_head = hk * p.G + p.G * split / p.splits, heads = hk * p.G + p.G * (split + 1) / p.splits - first_head;
        tiles = heads * max(0, tb - ta);
    }
};

// Tiles of Q and dO (one behind the other in LDS) with the statistics of their rows, requested by NT threads.
template <int HD, bool DMA, int NT>
struct ColFeed {
    RowFeed<HD, DMA, NT> qf, gf;
    float stat;
    __device__ __forceinline__ ColFeed(const SeqParams& p, int tid) : qf(p.q.sl, p.D, tid), gf(p.g.sl, p.D, tid), stat(0.0f) {}
    __device__ __forceinline__ void request(const SeqParams& p, const SeqBlock& b, int hq, int r0, elem_t* place, int tid, int wave) {
        const int64_t token = b.token + r0;
        qf.request(p.q.head(0, hq) + token * p.q.sl, p.q.sl, b.tokens - r0, p.D, place, wave);
        gf.request(p.g.head(0, hq) + token * p.g.sl, p.g.sl, b.tokens - r0, p.D, place + SeqTile<HD>::kElems, wave);
        if (tid < 3 * kCtxTile) {
            const int i = tid & (kCtxTile - 1);
            const float* from = p.folded + (tid / kCtxTile * (int64_t)p.Hq + hq) * p.T + token;
            stat = r0 + i < b.tokens ? from[i] : tid < kCtxTile ? INFINITY : tid < 2 * kCtxTile ? 1.0f : 0.0f;
        }
    }
    __device__ __forceinline__ void deliver(const SeqParams& p, elem_t* place, float* stats, int tid) {
        qf.deliver(place, p.D, tid);
        gf.deliver(place + SeqTile<HD>::kElems, p.D, tid);
        if (tid < 3 * kCtxTile) stats[tid] = stat;
    }
};

// P and dS of 32 rows from their scores and dP - delta.  st: [row_stat_folded, -delta][64] from the first of the rows on; key: this lane's, from that row on.
template <bool MASKED, bool FACTORS>
__device__ __forceinline__ void col_probabilities(f32x16& s, f32x16& ds, const float* st, float c, int key, int h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 less = *reinterpret_cast<const f32x4*>(st + 8 * i + 4 * h);
        f32x4 factor;
        if constexpr (FACTORS) factor = *reinterpret_cast<const f32x4*>(st + kCtxTile + 8 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float y = fast_exp2(__builtin_fmaf(s[4 * i + j], c, -less[j]));
            if constexpr (FACTORS) y *= factor[j];
            ds[4 * i + j] *= y;
            if constexpr (MASKED)
                if (8 * i + j < key - 4 * h) y = 0.0f, ds[4 * i + j] = 0.0f;  // a row ahead of the key
            s[4 * i + j] = y;
        }
    }
}

// What is not finite of a tile of Q and dO: of the rows [first, end) to this lane's key, and out of the tile.
template <typename T, int HD, int NT>
__device__ __forceinline__ void col_care(f32x16* dk, f32x16* dv, elem_t* tile, int first, int end, int tid, int h) {
    add_not_finite<T, HD>(dk, tile, first, end, 0.0f, h);
    add_not_finite<T, HD>(dv, tile + SeqTile<HD>::kElems, first, end, 1.0f, h);
    workgroup_barrier();
    keep_finite<T, HD, NT>(tile, tid);
    keep_finite<T, HD, NT>(tile + SeqTile<HD>::kElems, tid);
    workgroup_barrier();
}

// dK or dV of a wave's 32 keys to where they go: the result, or a split's sums.
template <typename T, int HD>
__device__ __forceinline__ void store_col(const SeqParams& p, const SeqCols& w, f32x16* sum, bool some, float factor, const CtxView& out, int which, int k0,
                                          elem_t* region, int lane) {
    const int rows = min(max(w.b.tokens - k0, 0), 32);
    if (p.splits > 1) {
        const int64_t place = ((int64_t)(2 * w.split + which) * p.Hkv + w.hk) * p.T + w.b.token + k0;
        store_part<HD>(sum, some, p.part + place * HD, rows, lane);
    } else {
        store_rows_at<T, HD>(sum, some ? factor : 0.0f, rows, region, lane, p.D,
                             [&](int row) { return out.head(0, w.hk) + (int64_t)(w.b.token + k0 + row) * out.sl; });
    }
}

// Column-owned: four waves of 32 keys share tiles of 64 query rows, over all heads that read the key head (or, with splits, over a part of them).  Own K and V
// stay in registers.  64 sequences of 16 to 128 tokens, 12 heads, D=64, whole: 18.4 us = 2.3 TB/s, one tile to a workgroup.
template <typename T, int HD, bool DMA>
__global__ __launch_bounds__(kCtxThreads, 2) void seq_bwd_col(SeqParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = SeqTile<HD>::kElems, kHalf = 32 * SeqTile<HD>::kLd * 2, kBytes = SeqTile<HD>::kBytes;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);             // [2][Q, dO]
    float* stats = reinterpret_cast<float*>(tiles + 4 * kTile);  // [2][row_stat_folded, -delta][64]
    __shared__ int hurt;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const SeqCols w(p, lane);
    if (!w.b.some) return;
    const int keys = SeqKeys<false>(p, w.b).keys, k0 = w.b.row0 + 32 * wave, key = k0 + (lane & 31);
    const bool ok = key < keys;
    u32x4 own_k[HD / 16], own_v[HD / 16];
    own_operands<HD>(own_k, p.k.head(0, w.hk) + (int64_t)(w.b.token + key) * p.k.sl, ok, h, p.D);
    own_operands<HD>(own_v, p.v.head(0, w.hk) + (int64_t)(w.b.token + key) * p.v.sl, ok, h, p.D);
    ColFeed<HD, DMA, kCtxThreads> feed(p, tid);
    SeqTile<HD> at(tiles, lane);
    const auto place = [&](int x) { return tiles + (x & 1) * 2 * kTile; };
    const auto st_place = [&](int x) { return stats + (x & 1) * (kCtxStats / 2); };
    if (w.tiles) {
        feed.request(p, w.b, w.first_head, w.ta * kCtxTile, place(0), tid, wave);
        feed.deliver(p, place(0), st_place(0), tid);
        feed.qf.arrived();
    }
    f32x16 dk[HD / 32] = {}, dv[HD / 32] = {};
    int step = 2 * kBytes;
    if (tid == 0) hurt = 0;
    // x: tiles before this one; hq, t: the head and the tile of its rows
    const auto tile = [&](int x, int hq, int t, auto masked) {
        const int r0 = t * kCtxTile;
        const bool more = x + 1 < w.tiles;
        if (more) {
            const bool last = t + 1 == w.tb;
            feed.request(p, w.b, last ? hq + 1 : hq, (last ? w.ta : t + 1) * kCtxTile, place(x + 1), tid, wave);
        }
        const bool used = k0 < keys && !(decltype(masked)::value && r0 + kCtxTile <= k0);
        f32x16 s[2], ds[2];
        bool some = false;
        if (used) {
            const float* st = st_place(x);
            const bool factors = __builtin_amdgcn_ballot_w64(st[kCtxTile + lane] != 1.0f);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[u] = at.template scores<T>(u * kHalf, own_k);
                ds[u] = at.template scores<T>(kBytes + u * kHalf, own_v, seq_of_rows(st + 2 * kCtxTile + 32 * u, h));
            }
            if constexpr (decltype(masked)::value) some = some_not_finite(s[0], s[1]) || some_not_finite(ds[0], ds[1]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                constexpr bool kMasked = decltype(masked)::value;  // (factors may be NaN: ahead of the mask)
                col_probabilities<kMasked, kMasked>(s[u], ds[u], st + 32 * u, p.c, key - r0 - 32 * u, h);
                if (!kMasked && factors) {
                    const f32x16 factor = seq_of_rows(st + kCtxTile + 32 * u, h);
                    s[u] *= factor, ds[u] *= factor;
                }
            }
        }
        if constexpr (decltype(masked)::value)
            if (some_wave(&hurt, x, some, lane)) col_care<T, HD, kCtxThreads>(dk, dv, place(x), max(key - r0, 0), kCtxTile, tid, h);
        if (used) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                at.template add_columns<T>(dv, kBytes + u * kHalf, s[u]);
                at.template add_columns<T>(dk, u * kHalf, ds[u]);
            }
        }
        at.move(step);
        step = -step;
        if (more) feed.deliver(p, place(x + 1), st_place(x + 1), tid);
        feed.qf.arrived();
        workgroup_barrier();
    };
    workgroup_barrier();
    // causal: the rows of the block's own positions stand in a head's first two tiles
    const int near = p.causal ? min(kCtxOwned / kCtxTile, w.tb - w.ta) : 0;
    for (int done = 0, hq = w.first_head; done < w.tiles; ++hq) {
        int t = w.ta;
        for (; t < w.ta + near; ++t) tile(done++, hq, t, std::true_type{});
        for (; t < w.tb; ++t) tile(done++, hq, t, std::false_type{});
    }
    elem_t* region = tiles + wave * 32 * (HD + 8);
    store_col<T, HD>(p, w, dk, ok && keys != 1, p.scale, p.dk, 0, k0, region, lane);
    store_col<T, HD>(p, w, dv, ok, 1.0f, p.dv, 1, k0, region, lane);
}

// The same above D = 64, where the sums and operands of 32 keys are more than the registers of two waves to a SIMD: K and V stand in LDS, and a group
// of 32 keys has two waves, with 32 rows of a tile each, whose sums are added up in the end.  One workgroup to a compute unit (133 KB of LDS).  The
// sequences above at D=128: 655 us = 0.85 PFLOP/s, the matrix unit busy 44 %, LDS the most of the rest: five reads to two matrix instructions, none
// of which meets another in a bank.  (K and V in registers with eight waves: 982 us, spills.)
template <typename T, int HD, bool DMA>
__global__ __launch_bounds__(2 * kCtxThreads, 2) void seq_bwd_col_pair(SeqParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = SeqTile<HD>::kElems, kHalf = 32 * SeqTile<HD>::kLd * 2, kBytes = SeqTile<HD>::kBytes, NT = 2 * kCtxThreads;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);             // [2][Q, dO]
    elem_t* mine = tiles + 4 * kTile;                            // K [2], V [2]
    float* stats = reinterpret_cast<float*>(mine + 4 * kTile);   // [2][row_stat_folded, -delta][64]
    __shared__ int hurt;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int group = wave % kCtxWaves, half = wave / kCtxWaves;
    const SeqCols w(p, lane);
    if (!w.b.some) return;
    const int keys = SeqKeys<false>(p, w.b).keys, k0 = w.b.row0 + 32 * group, key = k0 + (lane & 31);
    const bool ok = key < keys;
    ColFeed<HD, DMA, NT> feed(p, tid);
    SeqTile<HD> at(tiles + half * (kHalf / 2), lane);  // (the second wave: rows 32 .. 63)
    const auto place = [&](int x) { return tiles + (x & 1) * 2 * kTile; };
    const auto st_place = [&](int x) { return stats + (x & 1) * (kCtxStats / 2); };
    if (w.tiles) {
        feed.request(p, w.b, w.first_head, w.ta * kCtxTile, place(0), tid, wave);
        feed.deliver(p, place(0), st_place(0), tid);
        RowFeed<HD, DMA, NT> kf(p.k.sl, p.D, tid), vf(p.v.sl, p.D, tid);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = w.b.row0 + i * kCtxTile;
            kf.request(p.k.head(0, w.hk) + (int64_t)(w.b.token + k) * p.k.sl, p.k.sl, keys - k, p.D, mine + i * kTile, wave);
            vf.request(p.v.head(0, w.hk) + (int64_t)(w.b.token + k) * p.v.sl, p.v.sl, keys - k, p.D, mine + (2 + i) * kTile, wave);
            kf.deliver(mine + i * kTile, p.D, tid);
            vf.deliver(mine + (2 + i) * kTile, p.D, tid);
        }
        feed.qf.arrived();
    }
    uint32_t own[HD / 16];  // LDS addresses of the wave's rows of K; V two tiles behind
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) own[c] = at.row[c] - half * kHalf + 4 * kBytes + group * kHalf;
    f32x16 dk[HD / 32] = {}, dv[HD / 32] = {};
    int step = 2 * kBytes;
    if (tid == 0) hurt = 0;
    const auto tile = [&](int x, int hq, int t, auto masked) {
        const int r0 = t * kCtxTile + 32 * half;  // the wave's rows
        const bool more = x + 1 < w.tiles;
        if (more) {
            const bool last = t + 1 == w.tb;
            feed.request(p, w.b, last ? hq + 1 : hq, (last ? w.ta : t + 1) * kCtxTile, place(x + 1), tid, wave);
        }
        const bool used = k0 < keys && !(decltype(masked)::value && r0 + 32 <= k0);
        f32x16 s = {}, ds;
        bool some = false;
        if (used) {
            const float* st = st_place(x) + 32 * half;
            ds = seq_of_rows(st + 2 * kCtxTile, h);
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                s = Mma32<T>::run(at.rows(0, c), *SeqTile<HD>::template at<const u32x4>(own[c]), s);
                ds = Mma32<T>::run(at.rows(kBytes, c), *SeqTile<HD>::template at<const u32x4>(own[c] + 2 * kBytes), ds);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // (-delta)
            reads_ahead<HD / 16, 4, 2, 1>();
            __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);  // (the other statistics)
            if constexpr (decltype(masked)::value) some = some_not_finite(s, ds);
            col_probabilities<decltype(masked)::value, true>(s, ds, st, p.c, key - r0, h);
        }
        if constexpr (decltype(masked)::value)
            if (some_wave(&hurt, x, some, lane)) col_care<T, HD, NT>(dk, dv, place(x), max(key - t * kCtxTile, 32 * half), 32 * half + 32, tid, h);
        if (used) {
            at.template add_columns<T>(dv, kBytes, s);
            at.template add_columns<T>(dk, 0, ds);
            reads_ahead<HD / 8, 2, 1, 2>();
        }
        at.move(step);
        step = -step;
        if (more) feed.deliver(p, place(x + 1), st_place(x + 1), tid);
        feed.qf.arrived();
        workgroup_barrier();
    };
    workgroup_barrier();
    const int near = p.causal ? min(kCtxOwned / kCtxTile, w.tb - w.ta) : 0;
    for (int done = 0, hq = w.first_head; done < w.tiles; ++hq) {
        int t = w.ta;
        for (; t < w.ta + near; ++t) tile(done++, hq, t, std::true_type{});
        for (; t < w.tb; ++t) tile(done++, hq, t, std::false_type{});
    }
    elem_t* region = tiles + group * 32 * (HD + 8);
    const auto finish = [&](f32x16* sum, bool some, float factor, const CtxView& out, int which) {
        // [group][register][lane]: the sums of the second waves take the place of the tiles
        f32x4* there = reinterpret_cast<f32x4*>(tiles) + group * (HD / 32) * 4 * 64 + lane;
        if (half)
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    there[(4 * dt + i) * 64] = f32x4{sum[dt][4 * i], sum[dt][4 * i + 1], sum[dt][4 * i + 2], sum[dt][4 * i + 3]};
        workgroup_barrier();
        if (!half)
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 other = there[(4 * dt + i) * 64];
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[dt][4 * i + j] += other[j];
                }
        workgroup_barrier();
        if (!half) store_col<T, HD>(p, w, sum, some, factor, out, which, k0, region, lane);
        workgroup_barrier();
    };
    finish(dk, ok && keys != 1, p.scale, p.dk, 0);
    finish(dv, ok, 1.0f, p.dv, 1);
}

// Adds up the splits of seq_bwd_col, eight columns to a thread, in a fixed order.  Two splits of 15000 tokens, four heads of 128: 154 MB in 23 us, from the caches in
// part.
template <typename T, int HD>
__global__ __launch_bounds__(kCtxThreads) void seq_sum(SeqParams p) {
    constexpr int CH = HD / 8;
    const int64_t x = (int64_t)blockIdx.x * kCtxThreads + threadIdx.x, rows = (int64_t)p.Hkv * p.T, place = x / CH;  // [dk, dv][Hkv][T]
    const int c8 = 8 * (int)(x % CH);
    if (place >= 2 * rows) return;
    float y[8] = {};
    for (int s = 0; s < p.splits; ++s) {
        const f32x4* from = reinterpret_cast<const f32x4*>(p.part + (2 * s * rows + place) * HD + c8);
        const f32x4 a = from[0], c = from[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += a[j], y[4 + j] += c[j];
    }
    const bool v = place >= rows;
    const int64_t row = v ? place - rows : place;
    const float f = v ? 1.0f : p.scale;
    const CtxView& out = v ? p.dv : p.dk;
    store_chunk(out.head(0, (int)(row / p.T)) + row % p.T * out.sl,
                u32x4{T::pack2(f * y[0], f * y[1]), T::pack2(f * y[2], f * y[3]), T::pack2(f * y[4], f * y[5]), T::pack2(f * y[6], f * y[7])}, c8, p.D);
}

}  // namespace sjvp
