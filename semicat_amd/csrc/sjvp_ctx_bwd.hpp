// Backward kernels of the attention on keys of another length / with a relative position bias (sjvp_ctx.hpp).
//
//   dP = dO V^T,  delta = rowsum(dO * O),  dS = P (dP - delta)
//   dQ = scale dS K,  dK = scale sum_heads dS^T Q,  dV = sum_heads P^T dO,  dtable[bucket][head] = sum of dS over its differences
//
// A row-owned launch (dQ, delta and the bucket sums) and a column-owned one (dK, dV), both of which recompute P: 3 + 4
// contractions against the 5 of a single launch, whose dQ would be summed over workgroups by atomics in an order that changes from run
// to run, except where a workgroup holds all keys of a sequence (ctx_bwd_one).
#pragma once
#include "sjvp_ctx.hpp"

namespace sjvp {

__device__ __forceinline__ float wave_sum(float x) {
    x = halves_sum(sum16(x));
    return x + __shfl_xor(x, 16);
}

// dO . (o + what its rounding left) over eight columns
template <typename T>
__device__ __forceinline__ float piece_delta(u32x4 g, u32x4 o, u32x4 rest) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 32; e += 16)
            sum += T::to_float((elem_t)(g[j] >> e)) * with_rest<T>((elem_t)(o[j] >> e), (elem_t)(rest[j] >> e));
    return sum;
}

// the same over the lane's own row, from the operands of dO
template <typename T, int HD>
__device__ __forceinline__ float row_delta(const CtxParams& p, const u32x4* own_g, const elem_t* o, const elem_t* rest, bool ok, int h) {
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) {
        if (!ok) continue;
        const u32x4 none = {0u, 0u, 0u, 0u};
        sum += piece_delta<T>(own_g[c], load_chunk(o, 16 * c + 8 * h, p.D), rest ? load_chunk(rest, 16 * c + 8 * h, p.D) : none);
    }
    return halves_sum(sum);
}

// What LDS holds of 32 looped rows, as the registers of a score tile.  -delta is where the contraction for dP starts, an instruction less to an
// element (B=8 Hq=16 Hkv=4 Lq=2048 Lk=1024 D=128 1.5 % of forward and backward), but not where dS is summed by bucket: the matrix unit cuts
// off what it adds below its larger addends, and the gradient of an fp32 table would be some 4e-6 off.
__device__ __forceinline__ f32x16 of_rows(const float* rows, int h) {
    f32x16 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 four = *reinterpret_cast<const f32x4*>(rows + 8 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = four[j];
    }
    return x;
}

// P and dS of 32 rows whose factors stand in LDS.
__device__ __forceinline__ void times_rows(f32x16& s, f32x16& ds, const float* rows, int h) {
    const f32x16 factors = of_rows(rows, h);
    s *= factors, ds *= factors;
}

// Sums along the diagonals of a 32 x 32 score tile (one wave's): lane j < 63 receives that of the difference (looped row - column)
// 31 - j.  The partial sum of a diagonal stands with the lane whose column it has reached and moves one lane up from a looped row to
// the next; the upper half of the wave, which holds columns of its own only until they are moved below it, takes what leaves the 32
// columns.  Registers and lane shifts alone.  (LDS atomics by difference took 190 cycles an instruction: B=64 H=12 L=128 D=64 160 us
// for the launch; through rows of LDS 35 us and 36 KB of it; this way 32 us.)
__device__ __forceinline__ float diagonals(const f32x16& x) {
    float lower[16], upper[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[r]), 0u, false, false);
        lower[r] = __uint_as_float(halves[0]);
        upper[r] = __uint_as_float(halves[1]);
    }
    float sum = 0.0f;
#pragma unroll
    for (int y = 0; y < 32; ++y) {
        const int r = 4 * (y >> 3) + (y & 3);
        sum = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(sum), 0x138, 0xf, 0xf, true)) + (y & 4 ? upper : lower)[r];
    }
    return sum;
}

// From a workgroup's sums by difference (`count` waves, one after another) to its sums by bucket: first over the waves, then by 16 lanes to
// a bucket.
__device__ __forceinline__ void write_buckets(const CtxParams& p, float* hists, int count, float* out, bool any, int tid, int threads) {
    const int nb = ctx_all_buckets(p), zero = p.far + kCtxPad, entries = ctx_row_entries(p);
    for (int x = tid; x < entries; x += threads) {
        float sum = hists[x];
        for (int k = 1; k < count; ++k) sum += hists[k * entries + x];
        hists[x] = sum;
    }
    workgroup_barrier();
    for (int bucket = tid / 16; bucket < (nb + 15) / 16 * 16; bucket += threads / 16) {
        const int side = bucket >= p.buckets, j = min(bucket - side * p.buckets, p.buckets - 1);
        const int from = p.first[j], to = j + 1 < p.buckets ? p.first[j + 1] - 1 : zero;  // distances
        const int lo = side ? zero + max(from, 1) : zero - to;
        const int hi = side ? zero + to : !p.both && from == 0 && to >= 0 ? entries - 1 : zero - from;  // (above zero: distance 0)
        float sum = 0.0f;
        for (int x = lo + (tid & 15); x <= hi; x += 16) sum += hists[x];
        sum = sum16(sum);
        if ((tid & 15) == 0 && bucket < nb) out[bucket] = any ? sum : 0.0f;
    }
}

// Row-owned: four waves of 32 query rows of one head share tiles of 64 keys.  Bound by the matrix unit and the vector instructions
// together with the latency of a tile, two waves to a SIMD: B=8 H=16 L=4096 D=64 causal with bias 530 us (three contractions at 0.78
// PFLOP/s, the matrix unit busy 37 %, vector instructions issued 56 %), B=8 Hq=16 Hkv=4 Lq=2048 Lk=1024 D=128 224 us.
template <typename T, int HD, bool BIAS, bool DMA>
__global__ __launch_bounds__(kCtxThreads, HD <= 64 && !BIAS ? 3 : 2) void ctx_bwd_row(CtxParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = Tile<HD, DMA>::kElems;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);  // [2][K, V]
    float* row = reinterpret_cast<float*>(tiles + 4 * kTile);
    const int nqb = p.blocks, entries = ctx_row_entries(p);
    const CtxWork w = ctx_work(p.B * p.Hkv, p.G * nqb * p.splits);
    if (!w.some) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int split = w.inner / (p.G * nqb), inner = w.inner % (p.G * nqb);
    const int b = w.unit / p.Hkv, hk = w.unit % p.Hkv, hq = hk * p.G + inner / nqb;
    const int qb = p.causal ? nqb - 1 - inner % nqb : inner % nqb;
    const CtxBatch bt(p, b);
    const int q0 = qb * kCtxOwned + 32 * wave, qi = q0 + (lane & 31);
    const int rows = min(max(bt.rows - q0, 0), 32), last = min(bt.rows, (qb + 1) * kCtxOwned) - 1;
    const int n = last >= qb * kCtxOwned ? bt.seen(p, last) : 0, n_wave = rows > 0 ? bt.seen(p, q0 + rows - 1) : 0;
    const int limit = bt.seen(p, qi), pos0 = bt.start + q0, pos = pos0 + (lane & 31);
    const int nt = (n + kCtxTile - 1) / kCtxTile;
    const int t0 = (int)((int64_t)nt * split / p.splits), t1 = (int)((int64_t)nt * (split + 1) / p.splits);
    float* hist = row + entries + wave * entries;  // the wave's sums of dS by difference

    const elem_t *kt = p.k.head(b, hk), *vt = p.v.head(b, hk);
    TileFeed<HD, DMA> kf(p.k.sl, p.D, tid), vf(p.v.sl, p.D, tid);
    const Tile<HD, DMA> at(lane);
    const auto place = [&](int t) { return tiles + ((t - t0) & 1) * 2 * kTile; };
    const auto request = [&](int t) {
        kf.request(kt + (int64_t)t * kCtxTile * p.k.sl, p.k.sl, n - t * kCtxTile, p.D, place(t), wave);
        vf.request(vt + (int64_t)t * kCtxTile * p.v.sl, p.v.sl, n - t * kCtxTile, p.D, place(t) + kTile, wave);
    };
    const auto deliver = [&](int t) {
        kf.deliver(place(t), p.D, tid);
        vf.deliver(place(t) + kTile, p.D, tid);
    };
    if (t0 < t1) request(t0);
    const int64_t stat = ((int64_t)b * p.Hq + hq) * p.Lq + qi;
    const bool mine = (lane & 31) < rows;
    const f32x2 ml = mine ? load_stat(p, stat) : f32x2{0.0f, 0.0f};
    u32x4 own_q[HD / 16], own_g[HD / 16];
    own_operands<HD>(own_q, p.q.head(b, hq) + (int64_t)qi * p.q.sl, mine, h, p.D);
    own_operands<HD>(own_g, p.g.head(b, hq) + (int64_t)qi * p.g.sl, mine, h, p.D);
    if constexpr (BIAS) {
        fill_bias_row(p, row, hq, tid, kCtxThreads);
        for (int x = lane; x < entries; x += 64) hist[x] = 0.0f;
    }
    const bool ok = ml[1] != 0.0f;         // a row that sees no key has no gradient, whatever its cotangent,
    const bool scored = ok && limit != 1;  // one that sees one key none of its score: exactly none, not what rounding leaves
    const f32x2 less_factor = row_stat(ml);
    const float less = less_factor[0], factor = less_factor[1];
    if (__builtin_amdgcn_ballot_w64(mine && !ok)) {
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) own_g[c] = ok ? own_g[c] : u32x4{0u, 0u, 0u, 0u};
    }
    const float delta = row_delta<T, HD>(p, own_g, p.o.head(b, hq) + (int64_t)qi * p.o.sl,
                                         p.rest.ptr ? p.rest.head(b, hq) + (int64_t)qi * p.rest.sl : nullptr, ok, h);
    if (split == 0 && h == 0 && qi < p.Lq) {
        const int64_t all = (int64_t)p.B * p.Hq * p.Lq;
        const f32x2 folded = row_stat_folded(ml);
        p.folded[stat] = folded[0], p.folded[all + stat] = folded[1], p.folded[2 * all + stat] = -delta;
    }
    const float less_delta = -delta * factor;  // P (dP - delta) = exponential * (factor dP + less_delta)
    if (t0 < t1) deliver(t0);
    kf.arrived();
    workgroup_barrier();
    // scores of 32 keys from k0 on to P without its factor, zero behind the sequence (masked)
    const auto exponentials = [&](f32x16& s, int k0, auto band, bool masked) {
        if constexpr (decltype(band)::value == kNear) {
            const float* bias = row + row_entry(p, k0 + 4 * h - pos, 28);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], p.c, bias[8 * (r >> 2) + (r & 3)]) - less);
        } else {
            const float one = BIAS ? row[band == kBelow ? 0 : entries - 1] - less : -less;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], p.c, one));
        }
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (tile_row(r, 0) >= bt.keys - k0 - 4 * h) s[r] = 0.0f;
        }
    };
    f32x16 acc[HD / 32] = {};
    float below = 0.0f, above = 0.0f;  // sums of dS beyond the last single distance
    // (the sequence's last tile with its mask in code of its own, as in the forward)
    const auto tile = [&](int t, bool masked, auto band) {
        const int key = t * kCtxTile;
        if (t + 1 < t1) request(t + 1);
        const elem_t* K = place(t);
        if (key < n_wave) {
            f32x16 s[2], ds[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[u] = scores<T>(at, K, 32 * u, own_q);
                ds[u] = scores<T>(at, K + kTile, 32 * u, own_g);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                exponentials(s[u], key + 32 * u, band, masked);
#pragma unroll
                for (int r = 0; r < 16; ++r) ds[u][r] = s[u][r] * __builtin_fmaf(ds[u][r], factor, less_delta);
                if constexpr (BIAS && decltype(band)::value == kNear) {
                    const float sum = diagonals(ds[u]);
                    if (lane < 63) hist[row_entry(p, key + 32 * u - pos0 - 31, 63) + 62 - lane] += sum;
                    wave_exchange();  // (other lanes add to these next)
                } else if constexpr (BIAS) {
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += ds[u][r];
                    if constexpr (decltype(band)::value == kBelow) below += sum;
                    else above += sum;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) add_columns<T>(acc, at, K, 32 * u, ds[u]);
        }
        if (t + 1 < t1) deliver(t + 1);
        kf.arrived();
        workgroup_barrier();
    };
    // the tiles near the diagonal of the workgroup, whose positions are first .. first + 127
    const int first = bt.start + qb * kCtxOwned;
    const int whole = t1 * kCtxTile > bt.keys ? t1 - 1 : t1;
    int t = t0;
    if constexpr (BIAS) {
        const int t_near = ctx_rounds(row[0]) ? 0 : tiles_before(first - p.far + 1, nt);
        const int t_above = ctx_rounds(row[entries - 1]) ? nt : tiles_before(first + kCtxOwned - 1 + p.far + kCtxTile - 1, nt);
        for (; t < min(t_near, whole); ++t) tile(t, false, InBand<kBelow>{});
        for (; t < min(t_above, whole); ++t) tile(t, false, InBand<kNear>{});
        for (; t < whole; ++t) tile(t, false, InBand<kAbove>{});
    } else {
        for (; t < whole; ++t) tile(t, false, InBand<kBelow>{});
    }
    // (differences beyond the last single distance may be summed among the others, at the row's ends)
    if (t < t1) tile(t, true, InBand<BIAS ? kNear : kBelow>{});
    const int out_rows = min(max(p.Lq - q0, 0), 32);
    if (p.splits > 1) {
        const int64_t all = (int64_t)p.B * p.Hq * p.Lq;
        store_part<HD>(acc, scored, p.part + (split * all + ((int64_t)b * p.Hq + hq) * p.Lq + q0) * HD, out_rows, lane);
    } else {
        store_rows<T, HD>(acc, scored ? p.scale : 0.0f, p.dq.head(b, hq) + (int64_t)q0 * p.dq.sl, p.dq.sl, out_rows,
                          tiles + wave * 32 * (HD + 8), lane, p.D);
    }
    if constexpr (BIAS) {
        if (!p.tpart) return;
        below = wave_sum(below), above = wave_sum(above);
        if (lane == 0) hist[0] += below, hist[entries - 1] += above;
        workgroup_barrier();
        write_buckets(p, row + entries, kCtxWaves, p.tpart + (((int64_t)hq * p.B + b) * nqb * p.splits + (int64_t)qb * p.splits + split) * ctx_all_buckets(p),
                      bt.any_scored(p), tid, kCtxThreads);
    }
}

// Column-owned: four waves of 32 keys share tiles of 64 query rows, over all heads that read the key head.  Bound as the row-owned
// launch, at D = 128 with one wave to a SIMD (dK, dV, K and V of a wave are 256 registers): the cases above 640 us (four
// contractions at 0.86 PFLOP/s) and 310 us.  (Half tiles in a rolled loop: 1 % and 4 % slower.)
template <typename T, int HD, bool BIAS, bool DMA>
__global__ __launch_bounds__(kCtxThreads, HD <= 64 ? 2 : 1) void ctx_bwd_col(CtxParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = Tile<HD, DMA>::kElems;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);                // [2][Q, dO]
    float* stats = reinterpret_cast<float*>(tiles + 4 * kTile);     // [2][row_stat_folded, -delta][64]
    float* bias_row = stats + kCtxStats;
    const int nkb = p.blocks, entries = ctx_row_entries(p);
    const CtxWork w = ctx_work(p.B * p.Hkv, nkb * p.splits);
    if (!w.some) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int split = w.inner / nkb, kb = w.inner % nkb;
    const int b = w.unit / p.Hkv, hk = w.unit % p.Hkv;
    const CtxBatch bt(p, b);
    const int k0 = kb * kCtxOwned + 32 * wave, key = k0 + (lane & 31);
    const bool ok = key < bt.keys;
    u32x4 own_k[HD / 16], own_v[HD / 16];
    own_operands<HD>(own_k, p.k.head(b, hk) + (int64_t)key * p.k.sl, ok, h, p.D);
    own_operands<HD>(own_v, p.v.head(b, hk) + (int64_t)key * p.v.sl, ok, h, p.D);
    // tiles of query rows that see a key of the workgroup
    const int first_row = p.causal ? max(0, kb * kCtxOwned - bt.start) : 0;
    const int ta = first_row / kCtxTile, tb = (bt.rows + kCtxTile - 1) / kCtxTile;
    const int per_head = kb * kCtxOwned < bt.keys ? max(0, tb - ta) : 0;
    const int64_t all = (int64_t)p.G * per_head;
    const int x0 = (int)(all * split / p.splits), x1 = (int)(all * (split + 1) / p.splits);

    TileFeed<HD, DMA> qf(p.q.sl, p.D, tid), gf(p.g.sl, p.D, tid);
    const Tile<HD, DMA> at(lane);
    float stat = 0.0f;
    const auto place = [&](int x) { return tiles + ((x - x0) & 1) * 2 * kTile; };
    const auto request = [&](int x) {
        const int hq = hk * p.G + x / per_head, r0 = (ta + x % per_head) * kCtxTile;
        qf.request(p.q.head(b, hq) + (int64_t)r0 * p.q.sl, p.q.sl, bt.rows - r0, p.D, place(x), wave);
        gf.request(p.g.head(b, hq) + (int64_t)r0 * p.g.sl, p.g.sl, bt.rows - r0, p.D, place(x) + kTile, wave);
        if (tid < 3 * kCtxTile) {
            const int i = r0 + (tid & (kCtxTile - 1));
            const float* from = p.folded + ((tid / kCtxTile * (int64_t)p.B + b) * p.Hq + hq) * p.Lq;
            stat = i < bt.rows ? from[i] : tid < kCtxTile ? INFINITY : tid < 2 * kCtxTile ? 1.0f : 0.0f;
        }
    };
    const auto deliver = [&](int x) {
        qf.deliver(place(x), p.D, tid);
        gf.deliver(place(x) + kTile, p.D, tid);
        if (tid < 3 * kCtxTile) stats[((x - x0) & 1) * (kCtxStats / 2) + tid] = stat;
    };
    if (x0 < x1) {
        request(x0);
        deliver(x0);
        qf.arrived();
    }
    f32x16 dk[HD / 32] = {}, dv[HD / 32] = {};
    // The rows' factors (row_stat_folded) in every tile, or by a branch: B=8 Hq=16 Hkv=4 Lq=2048 Lk=1024 D=128 forward and backward 673 / 689 us;
    // at D = 64 B=8 H=16 L=1024 196 / 192.5, causal L=4096 with bias 1776 / 1754.
    constexpr bool kFactors = HD > 64;
    const auto tile = [&](int x, auto band) {
        const int p0 = bt.start + (ta + x % per_head) * kCtxTile;  // position of the first row
        if (x + 1 < x1) request(x + 1);
        const elem_t* Q = place(x);
        const float* st = stats + ((x - x0) & 1) * (kCtxStats / 2);
        if (k0 < bt.keys) {
            const bool factors = __builtin_amdgcn_ballot_w64(st[kCtxTile + lane] != 1.0f);
            f32x16 s[2], ds[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[u] = scores<T>(at, Q, 32 * u, own_k);
                ds[u] = scores<T>(at, Q + kTile, 32 * u, own_v, of_rows(st + 2 * kCtxTile + 32 * u, h));
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float* bias = bias_row;
                float one = 0.0f;
                if constexpr (BIAS && decltype(band)::value == kNear)
                    bias += row_entry(p, key - p0 - 32 * u - 4 * h - 27, 28) + 27;
                else if constexpr (BIAS) one = bias_row[band == kBelow ? 0 : entries - 1];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 less = *reinterpret_cast<const f32x4*>(st + 32 * u + 8 * i + 4 * h);
                    f32x4 factor;
                    if constexpr (kFactors) factor = *reinterpret_cast<const f32x4*>(st + kCtxTile + 32 * u + 8 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float y = s[u][4 * i + j];
                        if constexpr (BIAS && decltype(band)::value == kNear) y = fast_exp2(__builtin_fmaf(y, p.c, bias[-(8 * i + j)]) - less[j]);
                        else y = fast_exp2(__builtin_fmaf(y, p.c, BIAS ? one - less[j] : -less[j]));
                        if constexpr (kFactors) y *= factor[j];
                        s[u][4 * i + j] = y;
                        ds[u][4 * i + j] *= y;
                    }
                }
            }
            if (!kFactors && factors) times_rows(s[0], ds[0], st + kCtxTile, h), times_rows(s[1], ds[1], st + kCtxTile + 32, h);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                add_columns<T>(dv, at, Q + kTile, 32 * u, s[u]);
                add_columns<T>(dk, at, Q, 32 * u, ds[u]);
            }
        }
        if (x + 1 < x1) deliver(x + 1);
        qf.arrived();
        workgroup_barrier();
    };
    // the rows of a head one after another: first those that lie far behind the keys, then those near them, then those far ahead
    const int kb0 = kb * kCtxOwned - bt.start;
    const int n_above = max(0, tiles_before(kb0 - p.far + 1, tb) - ta), n_near = max(n_above, tiles_before(kb0 + kCtxOwned - 1 + p.far + kCtxTile - 1, tb) - ta);
    if (!BIAS && x0 < x1) workgroup_barrier();
    for (int x = x0; x < x1;) {
        const int g = x / per_head, first = g * per_head, end = min(x1, first + per_head);
        if constexpr (BIAS) {
            // (every wave is behind the barrier of the last tile)
            fill_bias_row(p, bias_row, hk * p.G + g, tid, kCtxThreads);
            workgroup_barrier();
            const int above = ctx_rounds(bias_row[entries - 1]) ? 0 : n_above, near = ctx_rounds(bias_row[0]) ? per_head : n_near;
            for (; x < min(first + above, end); ++x) tile(x, InBand<kAbove>{});
            for (; x < min(first + near, end); ++x) tile(x, InBand<kNear>{});
        }
        for (; x < end; ++x) tile(x, InBand<kBelow>{});
    }
    const bool scored = ok && bt.any_scored(p);
    const int out_rows = min(max(p.Lk - k0, 0), 32);
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.B * p.Hkv * p.Lk, place = ((int64_t)b * p.Hkv + hk) * p.Lk + k0;
        store_part<HD>(dk, scored, p.part + (2 * split * rows + place) * HD, out_rows, lane);
        store_part<HD>(dv, ok, p.part + ((2 * split + 1) * rows + place) * HD, out_rows, lane);
    } else {
        elem_t* region = tiles + wave * 32 * (HD + 8);
        store_rows<T, HD>(dk, scored ? p.scale : 0.0f, p.dk.head(b, hk) + (int64_t)k0 * p.dk.sl, p.dk.sl, out_rows, region, lane, p.D);
        store_rows<T, HD>(dv, ok ? 1.0f : 0.0f, p.dv.head(b, hk) + (int64_t)k0 * p.dv.sl, p.dv.sl, out_rows, region, lane, p.D);
    }
}

// One launch for both, where a workgroup's waves own all keys of a sequence between them (up to 32 * WAVES; head dimensions 33 to
// 64): five contractions, and each input is read once.  Column-owned as above; a tile's dS goes to LDS as well, where the dQ of the
// tile's rows is contracted over all keys, by a quarter of 32 rows x 32 columns for each of four waves.  With eight waves the two
// halves of the workgroup take turns, and the other half is ahead with the next tile's scores meanwhile; where two tiles' dS fit LDS, they
// alternate, which leaves one barrier to a tile (B=64 H=12 1024 x 256 with bias 305 us, with one 314).
// B=128 H=12 L=256 D=64 with bias 212 us against 132 row-owned + 125 column-owned, B=64 H=12 L=128 48 against 32.5 + 27.5.  Bound by
// the latency of a tile's chain (scores, dS to LDS, barrier, dQ): one workgroup of eight waves to a compute unit, vector instructions
// issued 38 % of the time, the matrix unit busy 13 %.
template <typename T, bool BIAS, bool DMA, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void ctx_bwd_one(CtxParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int HD = 64, NT = 64 * WAVES, kTile = Tile<HD, DMA>::kElems, kX = Tile<HD, false>::kElems;
    elem_t* const K = reinterpret_cast<elem_t*>(smem);                   // [WAVES / 2] tiles of all keys
    elem_t* const tiles = K + WAVES / 2 * kTile;                         // [2][Q, dO]
    elem_t* const X = tiles + 4 * kTile;                                 // [sets][WAVES / 2] tiles of dS, rows: keys, columns: query rows
    const int sets = WAVES == 8 ? p.packed : 1;
    float* const stats = reinterpret_cast<float*>(X + sets * (WAVES / 2) * kX);  // [2][row_stat_folded, -delta][64]
    float* const bias_row = stats + kCtxStats;                           // with 28 entries of -inf behind it
    const int entries = ctx_row_entries(p);
    float* const hists = bias_row + entries + 28;
    const CtxWork w = ctx_work(p.B * p.Hkv, 1);
    if (!w.some) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int b = w.unit / p.Hkv, hk = w.unit % p.Hkv;
    const CtxBatch bt(p, b);
    const int k0 = 32 * wave, key = k0 + (lane & 31);
    const bool ok = key < bt.keys;
    const int per_head = (p.Lq + kCtxTile - 1) / kCtxTile, all = p.G * per_head;
    float* const hist = hists + wave * entries;

    TileFeed<HD, DMA, NT> qf(p.q.sl, p.D, tid), gf(p.g.sl, p.D, tid), kf(p.k.sl, p.D, tid);
    const Tile<HD, DMA> at(lane);
    const Tile<HD, false> x_at(lane);
    // The statistics of a tile's rows: WAVES lanes to a row, each with every WAVES-th piece of dO, o and its rest.
    constexpr int kPieces = HD / 8 / WAVES;
    u32x4 g_piece[kPieces], o_piece[kPieces], r_piece[kPieces];
    f32x2 stat_next = {};
    const auto place = [&](int x) { return tiles + (x & 1) * 2 * kTile; };
    const auto request = [&](int x) {
        const int hq = hk * p.G + x / per_head, r0 = x % per_head * kCtxTile;
        qf.request(p.q.head(b, hq) + (int64_t)r0 * p.q.sl, p.q.sl, bt.rows - r0, p.D, place(x), wave);
        gf.request(p.g.head(b, hq) + (int64_t)r0 * p.g.sl, p.g.sl, bt.rows - r0, p.D, place(x) + kTile, wave);
        const int i = r0 + tid / WAVES;
        const bool mine = i < bt.rows;
        stat_next = mine ? load_stat(p, ((int64_t)b * p.Hq + hq) * p.Lq + i) : f32x2{0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int c8 = 8 * (tid % WAVES + WAVES * j);
            const u32x4 none = {0u, 0u, 0u, 0u};
            g_piece[j] = mine ? load_chunk(p.g.head(b, hq) + (int64_t)i * p.g.sl, c8, p.D) : none;
            o_piece[j] = mine ? load_chunk(p.o.head(b, hq) + (int64_t)i * p.o.sl, c8, p.D) : none;
            r_piece[j] = mine && p.rest.ptr ? load_chunk(p.rest.head(b, hq) + (int64_t)i * p.rest.sl, c8, p.D) : none;
        }
    };
    const auto deliver = [&](int x) {
        qf.deliver(place(x), p.D, tid);
        gf.deliver(place(x) + kTile, p.D, tid);
        float delta = 0.0f;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) delta += piece_delta<T>(g_piece[j], o_piece[j], r_piece[j]);
        delta += lanes_turned<0xB1>(delta);  // lanes 1, 0, 3, 2 of four
        delta += lanes_turned<0x4E>(delta);  // 2, 3, 0, 1
        if (WAVES == 8) delta += lanes_turned<0x141>(delta);  // 7 .. 0 of eight
        if (tid % WAVES == 0) {
            float* st = stats + (x & 1) * (kCtxStats / 2) + tid / WAVES;
            const f32x2 stat = row_stat_folded(stat_next);
            st[0] = stat[0], st[kCtxTile] = stat[1];
            st[2 * kCtxTile] = -delta;
        }
    };
    for (int t = 0; t < WAVES / 2; ++t) {
        kf.request(p.k.head(b, hk) + (int64_t)t * kCtxTile * p.k.sl, p.k.sl, bt.keys - t * kCtxTile, p.D, K + t * kTile, wave);
        kf.deliver(K + t * kTile, p.D, tid);
    }
    request(0);
    u32x4 own_k[HD / 16], own_v[HD / 16];
    own_operands<HD>(own_k, p.k.head(b, hk) + (int64_t)key * p.k.sl, ok, h, p.D);
    own_operands<HD>(own_v, p.v.head(b, hk) + (int64_t)key * p.v.sl, ok, h, p.D);
    const auto new_head = [&](int hq) {
        fill_bias_row(p, bias_row, hq, tid, NT);
        for (int y = lane; y < entries; y += 64) hist[y] = 0.0f;
    };
    if constexpr (BIAS) {
        new_head(hk * p.G);  // (while the first tile is on its way)
        if (tid < 28) bias_row[entries + tid] = -INFINITY;
    }
    deliver(0);
    f32x16 dk[HD / 32] = {}, dv[HD / 32] = {};
    for (int x = 0; x < all; ++x) {
        const int hq = hk * p.G + x / per_head, r0 = x % per_head * kCtxTile, p0 = bt.start + r0;
        if (BIAS && r0 == 0 && x) new_head(hq);
        if (x == 0) qf.arrived();
        if (x == 0 || (BIAS && r0 == 0)) workgroup_barrier();
        if (x + 1 < all) request(x + 1);
        const elem_t* Q = place(x);
        const float* st = stats + (x & 1) * (kCtxStats / 2);
        const bool factors = __builtin_amdgcn_ballot_w64(st[kCtxTile + lane] != 1.0f);
        f32x16 s[2], ds[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = scores<T>(at, Q, 32 * u, own_k);
            if constexpr (BIAS) ds[u] = scores<T>(at, Q + kTile, 32 * u, own_v);
            else ds[u] = scores<T>(at, Q + kTile, 32 * u, own_v, of_rows(st + 2 * kCtxTile + 32 * u, h));
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // keys that do not exist have the bias -inf
            const float* bias = bias_row + (ok ? row_entry(p, key - p0 - 32 * u - 4 * h - 27, 28) : entries) + 27;
            const float one = ok ? 0.0f : -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 less = *reinterpret_cast<const f32x4*>(st + 32 * u + 8 * i + 4 * h);
                f32x4 less_delta = {};
                if constexpr (BIAS) less_delta = *reinterpret_cast<const f32x4*>(st + 2 * kCtxTile + 32 * u + 8 * i + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float y = s[u][4 * i + j];
                    if constexpr (BIAS) y = fast_exp2(__builtin_fmaf(y, p.c, bias[-(8 * i + j)]) - less[j]);
                    else y = fast_exp2(__builtin_fmaf(y, p.c, one - less[j]));
                    s[u][4 * i + j] = y;
                    ds[u][4 * i + j] = y * (BIAS ? ds[u][4 * i + j] + less_delta[j] : ds[u][4 * i + j]);
                }
            }
            if (factors) times_rows(s[u], ds[u], st + kCtxTile + 32 * u, h);
            if constexpr (BIAS) {
                const float sum = diagonals(ds[u]);  // (looped rows are the queries here)
                if (lane < 63) hist[row_entry(p, k0 - p0 - 32 * u - 31, 63) + lane] += sum;
                wave_exchange();
            }
        }
        if (sets == 1) workgroup_barrier();  // the last tile's dS has been read
        elem_t* const XT = X + (x & (sets - 1)) * (WAVES / 2) * kX;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<u32x2*>(XT + key * (HD + 8) + 32 * u + 8 * i + 4 * h) =
                    u32x2{T::pack2(ds[u][4 * i], ds[u][4 * i + 1]), T::pack2(ds[u][4 * i + 2], ds[u][4 * i + 3])};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            add_columns<T>(dv, at, Q + kTile, 32 * u, s[u]);
            add_columns<T>(dk, at, Q, 32 * u, ds[u]);
        }
        if (x + 1 < all) deliver(x + 1);
        qf.arrived();
        workgroup_barrier();
        if (WAVES == 4 || (wave >> 2) == (x & 1)) {
            const int dt = wave & 1, uq = wave >> 1 & 1, i = r0 + 32 * uq + (lane & 31);
            f32x16 dq = {};
            const int steps = (bt.keys + 15) / 16;
#pragma unroll 4
            for (int m = 0; m < steps; ++m)
                dq = Mma32<T>::run(at.columns(K + (m >> 2) * kTile, 16 * (m & 3), dt), x_at.columns(XT + (m >> 2) * kX, 16 * (m & 3), uq), dq);
            // a row that sees one key has no gradient of its score: exactly none, not what rounding leaves
            const float f = bt.seen(p, i) == 1 ? 0.0f : p.scale;
            if (i < p.Lq) {
                elem_t* out = p.dq.head(b, hq) + (int64_t)i * p.dq.sl;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    float z[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[j] = f == 0.0f ? 0.0f : dq[4 * y + j] * f;
                    store_quad(out, u32x2{T::pack2(z[0], z[1]), T::pack2(z[2], z[3])}, 32 * dt + 8 * y + 4 * h, p.D);
                }
            }
        }
        if (BIAS && p.tpart && r0 + kCtxTile >= p.Lq) {
            write_buckets(p, hists, WAVES, p.tpart + ((int64_t)hq * p.B + b) * ctx_all_buckets(p), bt.any_scored(p), tid, NT);
            workgroup_barrier();
        }
    }
    workgroup_barrier();
    const bool scored = ok && bt.any_scored(p);
    const int out_rows = min(max(p.Lk - k0, 0), 32);
    elem_t* region = X + wave * 32 * (HD + 8);
    store_rows<T, HD>(dk, scored ? p.scale : 0.0f, p.dk.head(b, hk) + (int64_t)k0 * p.dk.sl, p.dk.sl, out_rows, region, lane, p.D);
    store_rows<T, HD>(dv, ok ? 1.0f : 0.0f, p.dv.head(b, hk) + (int64_t)k0 * p.dv.sl, p.dv.sl, out_rows, region, lane, p.D);
}

// Adds up the splits of a launch above: one thread to eight columns of a row of dQ, or of dK and dV.
template <typename T, int HD>
__global__ __launch_bounds__(kCtxThreads) void ctx_sum(CtxParams p) {
    constexpr int CH = HD / 8;
    const int H = p.cols ? p.Hkv : p.Hq, L = p.cols ? p.Lk : p.Lq, tensors = p.cols ? 2 : 1;
    const int64_t rows = (int64_t)p.B * H * L, x = (int64_t)blockIdx.x * kCtxThreads + threadIdx.x, place = x / CH;
    if (place >= tensors * rows) return;
    const int c8 = 8 * (int)(x % CH), second = place >= rows;
    f32x4 a = {}, c = {};
    for (int s = 0; s < p.splits; ++s) {
        const float* from = p.part + (s * tensors * rows + place) * HD + c8;
        a += *reinterpret_cast<const f32x4*>(from);
        c += *reinterpret_cast<const f32x4*>(from + 4);
    }
    const int64_t at = place - second * rows, head = at / L;
    const CtxView& out = !p.cols ? p.dq : second ? p.dv : p.dk;
    const float f = second ? 1.0f : p.scale;
    const u32x4 y = {T::pack2(a[0] * f, a[1] * f), T::pack2(a[2] * f, a[3] * f), T::pack2(c[0] * f, c[1] * f), T::pack2(c[2] * f, c[3] * f)};
    store_chunk(out.head((int)(head / H), (int)(head % H)) + (at % L) * out.sl, y, c8, p.D);
}

}  // namespace sjvp
