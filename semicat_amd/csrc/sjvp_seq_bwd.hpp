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

// Row-owned: four waves of 32 query rows (of the heads that share a key head) share tiles of 64 keys.
template <typename T, int HD, bool DMA>
__global__ __launch_bounds__(kCtxThreads, HD <= 64 ? 3 : 2) void seq_bwd_row(SeqParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = SeqTile<HD>::kElems;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);  // K [2], V [2]
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
        const bool more = t + 1 < nt;
        if (more) feed.request(p, t + 1, n, k_place(t + 1), v_place(t + 1), wave);
        if (key < n_wave) {
            f32x16 s[2], ds[2];
            s[0] = s[1] = ds[0] = ds[1] = f32x16{};
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    s[u] = Mma32<T>::run(at.rows(u * kHalf, c), own_q[c], s[u]);
                    ds[u] = Mma32<T>::run(at.rows(2 * kBytes + u * kHalf, c), own_g[c], ds[u]);
                }
            reads_ahead<HD / 8, 2, 2, 2>();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    ds[u][r] = fast_exp2(__builtin_fmaf(s[u][r], p.c, -less)) * __builtin_fmaf(ds[u][r], factor, less_delta);
                    if constexpr (decltype(masked)::value)
                        if (32 * u + tile_row(r, 0) >= limit - key - 4 * h) ds[u][r] = 0.0f;
                }
                at.template add_columns<T>(acc, u * kHalf, ds[u]);
            }
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

// Column-owned: groups of 32 keys share tiles of 64 query rows, over all heads that read the key head (or, with splits, over a part of them).  A group is
// one wave, or two that take 32 rows of a tile each and add their sums up in the end: at D = 128 the sums and operands of 32 keys fill the
// registers of two waves to a SIMD either way, and two waves fill each other's gaps.
template <typename T, int HD, bool DMA, int PAIR>
__global__ __launch_bounds__(kCtxThreads * PAIR, HD <= 64 ? 2 * PAIR : PAIR) void seq_bwd_col(SeqParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = SeqTile<HD>::kElems, NT = kCtxThreads * PAIR, U = 2 / PAIR;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);             // [2][Q, dO]
    elem_t* mine = tiles + 4 * kTile;                            // PAIR == 2: K [2], V [2] of the workgroup's keys
    float* stats = reinterpret_cast<float*>(mine + (PAIR == 2 ? 4 * kTile : 0));  // [2][row_stat_folded, -delta][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int group = wave % kCtxWaves, half = wave / kCtxWaves;
    const int hk = blockIdx.x % p.Hkv, x = blockIdx.x / p.Hkv, split = x % p.splits;  // (splits side by side: they are equally long)
    const SeqBlock b = seq_block_long_first<kCtxOwned>(p, x / p.splits, 1, true, lane);
    if (!b.some) return;
    const SeqKeys<false> keys(p, b);
    const int k0 = b.row0 + 32 * group, key = k0 + (lane & 31);
    const bool ok = key < keys.keys;
    u32x4 own_k[PAIR == 1 ? HD / 16 : 1], own_v[PAIR == 1 ? HD / 16 : 1];
    if constexpr (PAIR == 1) {
        own_operands<HD>(own_k, p.k.head(0, hk) + (int64_t)(b.token + key) * p.k.sl, ok, h, p.D);
        own_operands<HD>(own_v, p.v.head(0, hk) + (int64_t)(b.token + key) * p.v.sl, ok, h, p.D);
    }
    // tiles of query rows that see a key of the workgroup, head by head
    const int ta = p.causal ? b.row0 / kCtxTile : 0, tb = (keys.keys + kCtxTile - 1) / kCtxTile, per_head = max(0, tb - ta);
    const int first_head = hk * p.G + p.G * split / p.splits, heads = hk * p.G + p.G * (split + 1) / p.splits - first_head;
    const int nx = heads * per_head;

    RowFeed<HD, DMA, NT> qf(p.q.sl, p.D, tid), gf(p.g.sl, p.D, tid);
    constexpr int kHalf = 32 * SeqTile<HD>::kLd * 2, kBytes = SeqTile<HD>::kBytes;
    SeqTile<HD> at(tiles + (PAIR == 2 ? half * (kHalf / 2) : 0), lane);  // (a pair's second wave: rows 32 .. 63)
    float stat = 0.0f;
    const auto place = [&](int x) { return tiles + (x & 1) * 2 * kTile; };
    const auto request = [&](int x, int hq, int r0) {
        const int64_t token = b.token + r0;
        qf.request(p.q.head(0, hq) + token * p.q.sl, p.q.sl, b.tokens - r0, p.D, place(x), wave);
        gf.request(p.g.head(0, hq) + token * p.g.sl, p.g.sl, b.tokens - r0, p.D, place(x) + kTile, wave);
        if (tid < 3 * kCtxTile) {
            const int i = tid & (kCtxTile - 1);
            const float* from = p.folded + (tid / kCtxTile * (int64_t)p.Hq + hq) * p.T + token;
            stat = r0 + i < b.tokens ? from[i] : tid < kCtxTile ? INFINITY : tid < 2 * kCtxTile ? 1.0f : 0.0f;
        }
    };
    const auto deliver = [&](int x) {
        qf.deliver(place(x), p.D, tid);
        gf.deliver(place(x) + kTile, p.D, tid);
        if (tid < 3 * kCtxTile) stats[(x & 1) * (kCtxStats / 2) + tid] = stat;
    };
    if (nx) {
        request(0, first_head, ta * kCtxTile);
        deliver(0);
        if constexpr (PAIR == 2) {
            RowFeed<HD, DMA, NT> kf(p.k.sl, p.D, tid), vf(p.v.sl, p.D, tid);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int k = b.row0 + i * kCtxTile;
                kf.request(p.k.head(0, hk) + (int64_t)(b.token + k) * p.k.sl, p.k.sl, keys.keys - k, p.D, mine + i * kTile, wave);
                vf.request(p.v.head(0, hk) + (int64_t)(b.token + k) * p.v.sl, p.v.sl, keys.keys - k, p.D, mine + (2 + i) * kTile, wave);
                kf.deliver(mine + i * kTile, p.D, tid);
                vf.deliver(mine + (2 + i) * kTile, p.D, tid);
            }
        }
        qf.arrived();
    }
    // scores of 32 rows of a tile and the wave's keys (32 group .. of the two tiles of K, or of V behind them)
    uint32_t own[HD / 16];
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) own[c] = at.row[c] - half * kHalf + 4 * kBytes + group * kHalf;
    const auto products = [&](int from, const u32x4* own_rows, int own_from, f32x16 x) {
        if constexpr (PAIR == 1) return at.template scores<T>(from, own_rows, x);
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) x = Mma32<T>::run(at.rows(from, c), *SeqTile<HD>::template at<const u32x4>(own[c] + own_from), x);
        return x;
    };
    f32x16 dk[HD / 32] = {}, dv[HD / 32] = {};
    constexpr bool kFactors = HD > 64;
    int step = 2 * kBytes;
    // x: tiles before this one; hq, t: the head and the tile of its rows
    const auto tile = [&](int x, int hq, int t, auto masked) {
        const int r0 = t * kCtxTile;
        if (x + 1 < nx) {
            const bool last = t + 1 == tb;
            request(x + 1, last ? hq + 1 : hq, (last ? ta : t + 1) * kCtxTile);
        }
        const float* st = stats + (x & 1) * (kCtxStats / 2);
        const bool factors = !kFactors && __builtin_amdgcn_ballot_w64(st[kCtxTile + lane] != 1.0f);
        const int row0 = PAIR == 2 ? 32 * half : 0, end = row0 + 32 * U;  // rows of the tile that are this wave's
        if (k0 < keys.keys && !(decltype(masked)::value && r0 + end <= k0)) {
            f32x16 s[U], ds[U];
            if constexpr (PAIR == 2) {
            s[0] = f32x16{};
            ds[0] = seq_of_rows(st + 2 * kCtxTile + row0, h);
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                s[0] = Mma32<T>::run(at.rows(0, c), *SeqTile<HD>::template at<const u32x4>(own[c]), s[0]);
                ds[0] = Mma32<T>::run(at.rows(kBytes, c), *SeqTile<HD>::template at<const u32x4>(own[c] + 2 * kBytes), ds[0]);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            reads_ahead<HD / 16, 4, 2, 1>();
            __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
            } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u] = products(u * kHalf, own_k, 0, f32x16{});
                ds[u] = products(kBytes + u * kHalf, own_v, 2 * kBytes, seq_of_rows(st + 2 * kCtxTile + row0 + 32 * u, h));
            }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float* sr = st + row0 + 32 * u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 less = *reinterpret_cast<const f32x4*>(sr + 8 * i + 4 * h);
                    f32x4 factor;
                    if constexpr (kFactors) factor = *reinterpret_cast<const f32x4*>(sr + kCtxTile + 8 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float y = fast_exp2(__builtin_fmaf(s[u][4 * i + j], p.c, -less[j]));
                        if constexpr (kFactors) y *= factor[j];
                        ds[u][4 * i + j] *= y;
                        if constexpr (decltype(masked)::value)
                            if (row0 + 32 * u + 8 * i + j < key - r0 - 4 * h) y = 0.0f, ds[u][4 * i + j] = 0.0f;  // a row ahead of the key
                        s[u][4 * i + j] = y;
                    }
                }
                if (!kFactors && factors) {
                    const f32x16 factor = seq_of_rows(sr + kCtxTile, h);
                    s[u] *= factor, ds[u] *= factor;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                at.template add_columns<T>(dv, kBytes + u * kHalf, s[u]);
                at.template add_columns<T>(dk, u * kHalf, ds[u]);
            }
            if constexpr (PAIR == 2) reads_ahead<HD / 8, 2, 1, 2>();
        }
        at.move(step);
        step = -step;
        if (x + 1 < nx) deliver(x + 1);
        qf.arrived();
        workgroup_barrier();
    };
    workgroup_barrier();
    // causal: the rows of the block's own positions stand in a head's first two tiles
    const int near = p.causal ? min(kCtxOwned / kCtxTile, per_head) : 0;
    for (int done = 0, hq = first_head; done < nx; ++hq) {
        int t = ta;
        for (; t < ta + near; ++t) tile(done++, hq, t, std::true_type{});
        for (; t < tb; ++t) tile(done++, hq, t, std::false_type{});
    }
    const bool scored = ok && keys.keys != 1;
    const int out_rows = min(max(b.tokens - k0, 0), 32);
    elem_t* region = tiles + group * 32 * (HD + 8);
    const auto finish = [&](f32x16* sum, bool some, float factor, const CtxView& out, int which) {
        if constexpr (PAIR == 2) {
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
        }
        if (half == 0) {
            if (p.splits > 1) {
                const int64_t place = ((int64_t)(2 * split + which) * p.Hkv + hk) * p.T + b.token + k0;
                store_part<HD>(sum, some, p.part + place * HD, out_rows, lane);
            } else {
                store_rows_at<T, HD>(sum, some ? factor : 0.0f, out_rows, region, lane, p.D,
                                     [&](int row) { return out.head(0, hk) + (int64_t)(b.token + k0 + row) * out.sl; });
            }
        }
        if constexpr (PAIR == 2) workgroup_barrier();
    };
    finish(dk, scored, p.scale, p.dk, 0);
    finish(dv, ok, 1.0f, p.dv, 1);
}

// Adds up the splits of seq_bwd_col, eight columns to a thread, in a fixed order.
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
