// Forward kernels of the attention on keys of another length / with a relative position bias (sjvp_ctx.hpp).
#pragma once
#include "sjvp_ctx.hpp"

namespace sjvp {

// One pass with the running maximum m and sum l of each row.  Scores are in units of log2.  The maximum that the exponentials
// refer to is only raised when a row's has grown by more than 2^8: until then the sums keep their scale, which 16-bit
// probabilities up to 2^8 and fp32 sums hold without loss, and the factors of the accumulators stay out of the loop.
template <int HD>
struct RowSums {
    f32x16 acc[HD / 32];
    float m, ref, l;  // maximum (-inf: no key yet), what is subtracted (finite), sum of this lane's half

    __device__ __forceinline__ RowSums() : acc{}, m(-INFINITY), ref(0.0f), l(0.0f) {}

    // Scores of 32 keys from `key` on with their bias.  row: the bias row of this lane's head; pos: the position of its query.
    __device__ __forceinline__ void bias(const CtxParams& p, f32x16& s, int key, int h, const float* row, int pos) const {
        const float* at = row + row_entry(p, key + 4 * h - pos, 28);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], p.c, at[8 * (r >> 2) + (r & 3)]);
    }

    // The rows' maxima with these scores.  EVEN: they have neither factor nor bias yet, and all have the bias `one`.  left: the
    // sequence's keys from the first of them on, where they do not fill the scores (masked).
    template <bool EVEN, int N>
    __device__ __forceinline__ void raise(const CtxParams& p, f32x16 (&s)[N], float one, int left, int h, bool masked) {
        if (masked) {
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * u + tile_row(r, 0) >= left - 4 * h) s[u][r] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int r = u ? 0 : 1; r < 16; ++r) top = fmaxf(top, s[u][r]);
        if constexpr (EVEN) top = __builtin_fmaf(top, p.c, one);
        if (__builtin_amdgcn_ballot_w64(top > m + 8.0f)) {
            const float grown = fmaxf(m, halves_max(top));
            const float now = grown == -INFINITY ? 0.0f : grown;
            const float f = m == -INFINITY ? 0.0f : fast_exp2(ref - now);
            m = grown, ref = now;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt) acc[dt] *= f;
        }
    }

    template <bool EVEN, int N>
    __device__ __forceinline__ void exponentials(const CtxParams& p, f32x16 (&s)[N], float one) {
        const float less = one - ref;
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = fast_exp2(EVEN ? __builtin_fmaf(s[u][r], p.c, less) : s[u][r] - ref);
                sum += s[u][r];
            }
        l += sum;
    }
};

// TERMS > 1, for a backward to follow: the gradients need delta = dO . o as it would be with unrounded probabilities (their sums over
// a row are differences of near numbers), so P goes into the contraction with what its rounding leaves, and so does o into memory.
// Two terms leave 2e-6 of o in bf16, for gradients that are rounded to 16 bits in the end.  The gradient of an fp32 table in bf16 takes
// three: a bucket's sum over all rows is far below its terms' where it all but cancels (in norm, B=H=1 L=300 D=128: 2.1e-6 of it off with two
// terms, 3.1e-7 with three), for 2 % of a training pass at L=256 D=64 and 8 % at a causal 4096.
//
// Many rows: four waves of 32 rows of one head share tiles of 64 keys.  Two tiles of K and V in LDS: the next one is on its way
// while this one is used, one barrier to a tile.  Bound by the issue of vector instructions and by power: of
// B=8 H=16 Lq=4096 Lk=1024 (half of the keys there) D=64, 141 us, vector instructions are issued 82 % of the time and the matrix unit is
// busy 47 %, at 1.7 GHz.  So the loops hold neither masks nor bounds, the running maximum is raised seldom, and up to D = 64 four
// waves share a SIMD (128 registers), whose instructions fill each other's gaps (141 us against 145 by two waves with the scores of the
// next tile ahead, in turn).
// At D = 128 two (B=8 Hq=16 Hkv=4 Lq=2048 Lk=1024 with rests: 196 us, the matrix unit busy 47 %).
template <typename T, int HD, bool BIAS, bool DMA, int TERMS>
__global__ __launch_bounds__(kCtxThreads, HD <= 64 ? 4 : 2) void ctx_fwd(CtxParams p) {
    if constexpr (DMA) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = Tile<HD, DMA>::kElems;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);  // K [2], V [2]
    float* row = reinterpret_cast<float*>(tiles + 4 * kTile);
    const int nqb = p.blocks;
    const CtxWork w = ctx_work(p.B * p.Hkv, p.G * nqb);
    if (!w.some) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int b = w.unit / p.Hkv, hk = w.unit % p.Hkv, hq = hk * p.G + w.inner / nqb;
    const int qb = p.causal ? nqb - 1 - w.inner % nqb : w.inner % nqb;  // causal: long rows first
    const CtxBatch bt(p, b);
    const int q0 = qb * kCtxOwned + 32 * wave;
    const int rows = min(max(bt.rows - q0, 0), 32), last = min(bt.rows, (qb + 1) * kCtxOwned) - 1;
    const int n = last >= qb * kCtxOwned ? bt.seen(p, last) : 0, n_wave = rows > 0 ? bt.seen(p, q0 + rows - 1) : 0;
    const int pos = bt.start + q0 + (lane & 31);

    u32x4 own[HD / 16];
    own_operands<HD>(own, p.q.head(b, hq) + (int64_t)(q0 + (lane & 31)) * p.q.sl, (lane & 31) < rows, h, p.D);
    const elem_t *kt = p.k.head(b, hk), *vt = p.v.head(b, hk);
    const int nt = (n + kCtxTile - 1) / kCtxTile;
    TileFeed<HD, DMA> kf(p.k.sl, p.D, tid), vf(p.v.sl, p.D, tid);
    const Tile<HD, DMA> at(lane);
    const auto k_place = [&](int t) { return tiles + (t & 1) * kTile; };
    const auto v_place = [&](int t) { return tiles + (2 + (t & 1)) * kTile; };
    const auto k_request = [&](int t) { kf.request(kt + (int64_t)t * kCtxTile * p.k.sl, p.k.sl, n - t * kCtxTile, p.D, k_place(t), wave); };
    const auto v_request = [&](int t) { vf.request(vt + (int64_t)t * kCtxTile * p.v.sl, p.v.sl, n - t * kCtxTile, p.D, v_place(t), wave); };
    const auto k_deliver = [&](int t) { kf.deliver(k_place(t), p.D, tid); };
    const auto v_deliver = [&](int t) { vf.deliver(v_place(t), p.D, tid); };
    if (nt) k_request(0), v_request(0);
    if constexpr (BIAS) fill_bias_row(p, row, hq, tid, kCtxThreads);
    if (nt) {
        k_deliver(0), v_deliver(0);
    }
    kf.arrived();
    workgroup_barrier();
    RowSums<HD> st;
    // The sequence's last tile may need a mask and has code of its own behind the loops (as a condition within, the compiler makes the
    // mask a select in every tile, a third of the vector instructions at D = 64).
    const auto tile = [&](int t, bool masked, bool more, auto band) {
        constexpr bool kEven = decltype(band)::value != kNear;
        const int key = t * kCtxTile;
        if (more) {
            k_request(t + 1);
            v_request(t + 1);
        }
        if (key < n_wave) {
            f32x16 s[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u] = scores<T>(at, k_place(t), 32 * u, own);
            const float one = !BIAS ? 0.0f : row[band == kBelow ? 0 : 2 * (p.far + kCtxPad)];
            if constexpr (!kEven) {
#pragma unroll
                for (int u = 0; u < 2; ++u) st.bias(p, s[u], key + 32 * u, h, row, pos);
            }
            st.template raise<kEven>(p, s, one, bt.keys - key, h, masked);
            st.template exponentials<kEven>(p, s, one);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if constexpr (TERMS > 1) add_columns_exact<T, TERMS>(st.acc, at, v_place(t), 32 * u, s[u]);
                else add_columns<T>(st.acc, at, v_place(t), 32 * u, s[u]);
            }
        }
        if (more) {
            k_deliver(t + 1);
            v_deliver(t + 1);
        }
        kf.arrived();
        workgroup_barrier();
    };
    if constexpr (BIAS) {
        const int first = bt.start + qb * kCtxOwned;
        const int near = ctx_rounds(row[0]) ? 0 : tiles_before(first - p.far + 1, nt - 1);
        const int above = ctx_rounds(row[2 * (p.far + kCtxPad)]) ? nt - 1 : tiles_before(first + kCtxOwned - 1 + p.far + kCtxTile - 1, nt - 1);
        int t = 0;
        for (; t < near; ++t) tile(t, false, true, InBand<kBelow>{});
        for (; t < above; ++t) tile(t, false, true, InBand<kNear>{});
        for (; t + 1 < nt; ++t) tile(t, false, true, InBand<kAbove>{});
    } else {
        for (int t = 0; t + 1 < nt; ++t) tile(t, false, true, InBand<kBelow>{});
    }
    if (nt) tile(nt - 1, nt * kCtxTile > bt.keys, false, InBand<BIAS ? kNear : kBelow>{});
    const int out_rows = min(max(p.Lq - q0, 0), 32);
    const float both = halves_sum(st.l), l = (lane & 31) < rows ? both : 0.0f;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (h == 0 && (lane & 31) < out_rows) store_stat(p, ((int64_t)b * p.Hq + hq) * p.Lq + q0 + lane, st.ref, l);
    elem_t* region = tiles + wave * 32 * (HD + 8);
    store_rows<T, HD>(st.acc, f, p.o.head(b, hq) + (int64_t)q0 * p.o.sl, p.o.sl, out_rows, region, lane, p.D);
    if constexpr (TERMS > 1)
        store_rows<T, HD>(st.acc, f, p.rest.head(b, hq) + (int64_t)q0 * p.rest.sl, p.rest.sl, out_rows, region, lane, p.D, true);
}

// Few rows: the query rows of all heads that share a key head stand in one block of 32 (row = head of the group * Lq + query), and
// waves share out the keys: each runs over tiles of 32 keys of its own, K straight from memory into the operand's registers, V through a
// region of LDS that no other wave reads, so that nothing but the end is synchronised.  The sums of the waves are
// joined in LDS; with several splits of the key axis they go to memory for ctx_join.  Bound by memory for many keys: 64 sequences of 1024 to
// 2048 keys, Hq=16 Hkv=4 D=128, 37 us of kernel at 5.4 TB/s; by latency otherwise (one query on 128 keys: 4.7 us).
// `packed` heads of a group stand in one block's rows: all of them, or one where their bias rows would not fit or a head
// fills a block by itself.
template <typename T, int HD, bool BIAS, int TERMS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, HD <= 64 ? 4 : 2) void ctx_fwd_few(CtxParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kRegion = 32 * (HD + 8), kSum = HD + 4;
    elem_t* region = reinterpret_cast<elem_t*>(smem);  // [WAVES] V tiles, then the waves' sums [WAVES][32][HD + 4] fp32
    float* sums = reinterpret_cast<float*>(smem);
    float* stats = sums + WAVES * 32 * kSum;       // [WAVES][32] maximum, then sum
    float* bias_rows = stats + 2 * WAVES * 32;
    const int packed = p.packed, groups = p.G / packed, all_rows = packed * p.Lq;
    const CtxWork w = ctx_work(p.B * p.Hkv * groups, p.blocks * p.splits);
    if (!w.some) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int b = w.unit / (p.Hkv * groups), hu = w.unit % (p.Hkv * groups), hk = hu / groups, hq0 = hu * packed;
    const int rb = w.inner % p.blocks, split = w.inner / p.blocks;
    const CtxBatch bt(p, b);
    const int r0 = rb * 32, rows = min(all_rows - r0, 32), r = r0 + (lane & 31);
    const int g = min(r, all_rows - 1) / p.Lq, i = min(r, all_rows - 1) % p.Lq, g0 = r0 / p.Lq;
    const bool mine = r < all_rows && i < bt.rows;
    // the queries of a block: consecutive ones of one head, or any where it holds the end of one
    const bool one_head = (r0 + rows - 1) / p.Lq == g0;
    const int i_first = one_head ? r0 % p.Lq : 0, i_last = one_head ? r0 % p.Lq + rows - 1 : p.Lq - 1;
    const int n = bt.rows > i_first ? bt.seen(p, min(i_last, bt.rows - 1)) : 0;
    const int pos = bt.start + i;
    const int tiles = (n + 31) / 32;
    const int t_first = (int)((int64_t)tiles * split / p.splits), t_end = (int)((int64_t)tiles * (split + 1) / p.splits);

    u32x4 own[HD / 16];
    own_operands<HD>(own, p.q.head(b, hq0 + g) + (int64_t)i * p.q.sl, mine, h, p.D);
    const elem_t *kp = p.k.head(b, hk), *vp = p.v.head(b, hk);
    constexpr int CH = HD / 8, NV = 32 * CH / 64;
    u32x4 kr[HD / 16], vr[NV];
    uint32_t ko[HD / 16], vo[NV];
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) ko[c] = chunk_offset(lane & 31, 16 * c + 8 * h, p.k.sl, p.D);
#pragma unroll
    for (int x = 0; x < NV; ++x) vo[x] = chunk_offset((lane + 64 * x) / CH, 8 * ((lane + 64 * x) % CH), p.v.sl, p.D);
    const auto load = [&](int t) {
        const int key = t * 32;
        const Rows kf = make_rows(kp + (int64_t)key * p.k.sl, p.k.sl, min(n - key, 32), p.D),
                   vf = make_rows(vp + (int64_t)key * p.v.sl, p.v.sl, min(n - key, 32), p.D);
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) kr[c] = read_chunk(kf, ko[c]);
#pragma unroll
        for (int x = 0; x < NV; ++x) vr[x] = read_chunk(vf, vo[x]);
    };
    int t = t_first + wave;
    if (t < t_end) load(t);
    const float* row = bias_rows;
    if constexpr (BIAS) {
        const int entries = ctx_row_entries(p), heads = (r0 + rows - 1) / p.Lq - g0 + 1;
        fill_bias_row(p, bias_rows, hq0 + g0, tid, 64 * WAVES, heads);
        row = bias_rows + (g - g0) * entries;
        workgroup_barrier();
    }
    RowSums<HD> st;
    elem_t* V = region + wave * kRegion;
    const Tile<HD, false> tile(lane);
    for (; t < t_end; t += WAVES) {
#pragma unroll
        for (int x = 0; x < NV; ++x) {
            const int at = lane + 64 * x;
            if (p.D % 8) vr[x] = chunk_shifted(vr[x], 8 * (at % CH), p.D);
            *reinterpret_cast<u32x4*>(V + (at / CH) * (HD + 8) + 8 * (at % CH)) = vr[x];
        }
        if (p.D % 8) {
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) kr[c] = chunk_shifted(kr[c], 16 * c + 8 * h, p.D);
        }
        f32x16 s[1] = {};
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) s[0] = Mma32<T>::run(kr[c], own[c], s[0]);
        if (t + WAVES < t_end) load(t + WAVES);
        const int key = t * 32;
        if constexpr (BIAS) st.bias(p, s[0], key, h, row, pos);
        st.template raise<!BIAS>(p, s, 0.0f, bt.keys - key, h, key + 32 > bt.keys);
        st.template exponentials<!BIAS>(p, s, 0.0f);
        wave_exchange();
        if constexpr (TERMS > 1) add_columns_exact<T, TERMS>(st.acc, tile, V, 0, s[0]);
        else add_columns<T>(st.acc, tile, V, 0, s[0]);
        wave_exchange();
    }
    const float l = halves_sum(st.l);
    workgroup_barrier();  // the sums take the place of the V tiles
    if (h == 0) {
        stats[wave * 32 + lane] = st.m == -INFINITY ? -INFINITY : st.ref;
        stats[(WAVES + wave) * 32 + lane] = l;
    }
    float* out = sums + (wave * 32 + (lane & 31)) * kSum + 4 * h;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4*>(out + 32 * dt + 8 * x) =
                f32x4{st.acc[dt][4 * x], st.acc[dt][4 * x + 1], st.acc[dt][4 * x + 2], st.acc[dt][4 * x + 3]};
    workgroup_barrier();
    for (int x = tid; x < 32 * CH; x += 64 * WAVES) {
        const int at = x / CH, c8 = 8 * (x % CH), rr = r0 + at;
        if (at >= rows) break;
        float top = -INFINITY, sum = 0.0f, y[8] = {};
#pragma unroll
        for (int k = 0; k < WAVES; ++k) top = fmaxf(top, stats[k * 32 + at]);
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            const float f = fast_exp2(stats[k * 32 + at] - ref);
            sum += f * stats[(WAVES + k) * 32 + at];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] += f * sums[(k * 32 + at) * kSum + c8 + j];
        }
        const int gg = rr / p.Lq, ii = rr % p.Lq, hq = hq0 + gg;
        const int64_t place = ((int64_t)b * p.Hq + hq) * p.Lq + ii;
        if (ii >= bt.rows) {
            sum = 0.0f, top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = 0.0f;
        }
        if (p.splits > 1) {
            const int64_t part = split * ((int64_t)p.B * p.Hq * p.Lq) + place;
            if (c8 == 0) p.stat[2 * part] = top, p.stat[2 * part + 1] = sum;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                *reinterpret_cast<f32x4*>(p.part + part * HD + c8 + 4 * j) = f32x4{y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]};
            continue;
        }
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (c8 == 0) store_stat(p, place, ref, sum);
        u32x4 o, rest;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = f == 0.0f ? 0.0f : y[2 * j] * f, c = f == 0.0f ? 0.0f : y[2 * j + 1] * f;
            o[j] = T::pack2(a, c);
            rest[j] = rest_of<T>(o[j], a, c);
        }
        store_chunk(p.o.head(b, hq) + (int64_t)ii * p.o.sl, o, c8, p.D);
        if constexpr (TERMS > 1) store_chunk(p.rest.head(b, hq) + (int64_t)ii * p.rest.sl, rest, c8, p.D);
    }
}

// Joins the splits of ctx_fwd_few: 16 threads to the columns of a row (eight each), `slices` of them to the splits, which meet in
// LDS.  (One thread over all splits: B=2 H=16 Lq=4 Lk=16385 D=128 in 64 splits 34 us.)
template <typename T, int HD>
__global__ __launch_bounds__(kCtxThreads) void ctx_join(CtxParams p) {
    __shared__ float met[kCtxThreads / 16][16][11];
    const int64_t all = (int64_t)p.B * p.Hq * p.Lq;
    const int slices = min(16, 1 << (32 - __builtin_clz(p.splits - 1))), group = threadIdx.x >> 4, slice = group % slices;
    const int64_t place = (int64_t)blockIdx.x * (16 / slices) + group / slices;
    const int c8 = 8 * (threadIdx.x & 15);
    const bool some = place < all && c8 < HD;
    float top = -INFINITY, sum = 0.0f, y[8] = {};
    const auto add = [&](float other_top, float other_sum, const float* other) {
        const float now = fmaxf(top, other_top), ref = now == -INFINITY ? 0.0f : now, f = fast_exp2(top - ref), g = fast_exp2(other_top - ref);
        top = now;
        sum = f * sum + g * other_sum;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = f * y[j] + g * other[j];
    };
    if (some) {
        for (int s = slice; s < p.splits; s += slices) {
            const int64_t part = s * all + place;
            const f32x4 a = *reinterpret_cast<const f32x4*>(p.part + part * HD + c8), c = *reinterpret_cast<const f32x4*>(p.part + part * HD + c8 + 4);
            const float other[8] = {a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
            add(p.stat[2 * part], p.stat[2 * part + 1], other);
        }
    }
    float* mine = met[group][threadIdx.x & 15];
    mine[0] = top, mine[1] = sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine[2 + j] = y[j];
    workgroup_barrier();
    if (slice || !some) return;
    for (int s = 1; s < slices; ++s) {
        const float* other = met[group + s][threadIdx.x & 15];
        add(other[0], other[1], other + 2);
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (c8 == 0) store_stat(p, place, top == -INFINITY ? 0.0f : top, sum);
    u32x4 o, rest;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = f == 0.0f ? 0.0f : y[2 * j] * f, c = f == 0.0f ? 0.0f : y[2 * j + 1] * f;
        o[j] = T::pack2(a, c);
        rest[j] = rest_of<T>(o[j], a, c);
    }
    const int64_t head = place / p.Lq;
    const int i = (int)(place % p.Lq), hq = (int)(head % p.Hq), b = (int)(head / p.Hq);
    store_chunk(p.o.head(b, hq) + (int64_t)i * p.o.sl, o, c8, p.D);
    if (p.rest.ptr) store_chunk(p.rest.head(b, hq) + (int64_t)i * p.rest.sl, rest, c8, p.D);
}

}  // namespace sjvp
