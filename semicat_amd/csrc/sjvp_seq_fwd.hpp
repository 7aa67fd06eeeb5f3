// Forward kernels of the attention over packed sequences and over a paged cache (sjvp_seq.hpp).
#pragma once
#include "sjvp_seq.hpp"

namespace sjvp {

// The rows of a block: those of all heads that share a key head, token by token (row = token * G + head of the group), so that they read their
// keys once and a short sequence fills a block.
struct SeqRow {
    int token, hq;  // token within the segment
    __device__ __forceinline__ SeqRow(const SeqParams& p, int hk, int row) : token(row / p.G), hq(hk * p.G + row % p.G) {}
};

// Many rows: four waves of 32 rows share tiles of 64 keys, two tiles of K and V in LDS, one barrier to a tile.
template <typename T, int HD, bool PAGED, typename FEED>
__global__ __launch_bounds__(kCtxThreads, HD <= 64 ? 4 : 2) void seq_fwd(SeqParams p) {
    if constexpr (FEED::kDma) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr bool DMA = FEED::kDma;
    constexpr int kTile = Tile<HD, DMA>::kElems;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);  // K [2], V [2]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % p.Hkv, slot = p.causal ? p.slots - 1 - (int)(blockIdx.x / p.Hkv) : blockIdx.x / p.Hkv;  // causal: long rows first
    const SeqBlock b = seq_block<kCtxOwned>(p, slot, p.G, lane);
    const int all = b.tokens * p.G;
    if (!b.some || all < p.least || all > p.most) return;
    const SeqKeys<PAGED> keys(p, b);
    const int r0 = b.row0 + 32 * wave, rows = min(max(all - r0, 0), 32);
    const SeqRow mine(p, hk, min(r0 + (lane & 31), all - 1));
    const bool ok = (lane & 31) < rows;
    const int limit = keys.seen(p, mine.token);
    const int n = keys.seen(p, (min(b.row0 + kCtxOwned, all) - 1) / p.G), whole = keys.seen(p, b.row0 / p.G);  // keys of the last, the first row
    const int n_wave = rows > 0 ? keys.seen(p, (r0 + rows - 1) / p.G) : 0;

    u32x4 own[HD / 16];
    own_operands<HD>(own, p.q.head(0, mine.hq) + (int64_t)(b.token + mine.token) * p.q.sl, ok, h, p.D);
    const int nt = (n + kCtxTile - 1) / kCtxTile;
    FEED feed(p, b, hk, tid);
    const Tile<HD, DMA> at(lane);
    const auto k_place = [&](int t) { return tiles + (t & 1) * kTile; };
    const auto v_place = [&](int t) { return tiles + (2 + (t & 1)) * kTile; };
    if (nt) {
        feed.look(p, 0, n);
        feed.request(p, 0, n, k_place(0), v_place(0), wave);
        if (nt > 1) feed.look(p, 1, n);
        feed.deliver(p, k_place(0), v_place(0), tid);
    }
    feed.arrived();
    workgroup_barrier();
    SeqSums<HD> st;
    const auto tile = [&](int t, auto masked) {
        const bool more = t + 1 < nt;
        if (more) {
            feed.request(p, t + 1, n, k_place(t + 1), v_place(t + 1), wave);
            if (t + 2 < nt) feed.look(p, t + 2, n);
        }
        if (t * kCtxTile < n_wave) {
            f32x16 s[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u] = scores<T>(at, k_place(t), 32 * u, own);
            st.template take<decltype(masked)::value>(s, p.c, limit - t * kCtxTile, h);
#pragma unroll
            for (int u = 0; u < 2; ++u) add_columns<T>(st.acc, at, v_place(t), 32 * u, s[u]);
        }
        if (more) feed.deliver(p, k_place(t + 1), v_place(t + 1), tid);
        feed.arrived();
        workgroup_barrier();
    };
    // (the tiles that all rows see as a whole have a loop without masks)
    const int free = min(whole / kCtxTile, nt);
    int t = 0;
    for (; t < free; ++t) tile(t, std::false_type{});
    for (; t < nt; ++t) tile(t, std::true_type{});
    const float both = halves_sum(st.l), l = limit > 0 ? both : 0.0f, f = l == 0.0f ? 0.0f : 1.0f / l;
    if (p.lse && h == 0 && ok)
        *reinterpret_cast<f32x2*>(p.lse + 2 * ((int64_t)mine.hq * p.T + b.token + mine.token)) = f32x2{l == 0.0f ? 0.0f : st.ref, l};
    store_rows_at<T, HD>(st.acc, f, rows, tiles + wave * 32 * (HD + 8), lane, p.D, [&](int row) {
        const SeqRow to(p, hk, r0 + row);
        return p.o.head(0, to.hq) + (int64_t)(b.token + to.token) * p.o.sl;
    });
}

// Splits of the tiles of 32 keys of a sequence: of kSeqLeast tiles or more, as many as the launch has at most.
constexpr int kSeqLeast = 16;
struct SeqSplit {
    int used, first, end;
    __device__ __forceinline__ SeqSplit(int tiles, int splits, int split) {
        const int per = max(kSeqLeast, (tiles + splits - 1) / splits);
        used = max(1, (tiles + per - 1) / per);
        first = min(split * per, tiles), end = min(first + per, tiles);
    }
};

// Where the sums of a row stand between seq_few and seq_join: by token, or, where seq_few serves the short sequences of a call alone
// (p.most is kSeqFew), by segment, kSeqFew rows to each.
__device__ __forceinline__ int64_t seq_group(const SeqParams& p) { return p.most == kSeqFew ? (int64_t)(p.B + 2) * kSeqFew : (int64_t)p.T * p.G; }
__device__ __forceinline__ int64_t seq_places(const SeqParams& p) { return p.Hkv * seq_group(p); }
__device__ __forceinline__ int64_t seq_place(const SeqParams& p, const SeqBlock& b, int hk, int row) {
    return hk * seq_group(p) + (p.most == kSeqFew ? (int64_t)b.segment * kSeqFew : (int64_t)b.token * p.G) + row;
}

// Few rows: 32 rows to a block and waves that share out its keys: each runs over tiles of 32 keys of its own, K straight from memory into
// the operand's registers, V through a region of LDS that no other wave reads, so that nothing but the end is synchronised.  The sums of
// the waves are joined in LDS; with several splits of the keys they go to memory for seq_join.
// E4M3: the cache's numbers have 8 bits; a lane's 16 bytes of K are the two halves of 32 columns then, and q is read in that order.
template <typename T, int HD, bool E4M3, int WAVES>
__global__ __launch_bounds__(64 * WAVES, HD <= 64 ? 4 : 2) void seq_few(SeqParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kRegion = 32 * (HD + 8), kSum = HD + 4, CH = HD / 8;
    elem_t* region = reinterpret_cast<elem_t*>(smem);  // [WAVES] V tiles, then the waves' sums [WAVES][32][HD + 4] fp32
    float* sums = reinterpret_cast<float*>(smem);
    float* stats = sums + WAVES * 32 * kSum;  // [WAVES][32] maximum, then sum
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % p.Hkv, x = blockIdx.x / p.Hkv, slot = x % p.slots, split = x / p.slots;
    const SeqBlock b = seq_block<32>(p, slot, p.G, lane);
    const int all = b.tokens * p.G;
    if (!b.some || all < p.least || all > p.most) return;
    const SeqKeys<true> keys(p, b);
    const int r0 = b.row0, rows = min(all - r0, 32);
    const SeqRow mine(p, hk, min(r0 + (lane & 31), all - 1));
    const int limit = keys.seen(p, mine.token), n = keys.seen(p, (r0 + rows - 1) / p.G), whole = keys.seen(p, r0 / p.G);
    const SeqSplit part((n + 31) / 32, p.splits, split);
    if (split >= part.used) return;

    u32x4 own[HD / 16];
    {
        const elem_t* q = p.q.head(0, mine.hq) + (int64_t)(b.token + mine.token) * p.q.sl;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
            const int c8 = E4M3 ? 32 * (c / 2) + 16 * h + 8 * (c % 2) : 16 * c + 8 * h;
            own[c] = (lane & 31) < rows ? load_chunk(q, c8, p.D) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    constexpr int NK = E4M3 ? HD / 32 : HD / 16, PC = E4M3 ? HD / 16 : CH, NV = 32 * PC / 64;  // 16-byte pieces: K of a lane, V of a row, V of a lane
    u32x4 kr[NK], vr[NV];
    uint32_t ks[E4M3 ? NK : 1], vs[E4M3 ? NV : 1];
    const int* table = p.pages.table + (b.segment - 1) * p.pages.table_stride;
    const int64_t head = hk * p.pages.sh, scale_head = hk * p.pages.scale_sh;
    const void* none = &kZeroPiece;
    // the page of key t * 32 + lane % 32
    const auto look = [&](int t) {
        const int key = 32 * t + (lane & 31);
        return key < n ? table[p.pages.page_of(key)] : -1;
    };
    const auto load = [&](int t, int page) {
        const int key = 32 * t + (lane & 31), row = key - p.pages.page_of(key) * p.pages.size;
        const bool there = (uint32_t)page < (uint32_t)p.pages.pages;
        const int64_t at = page * p.pages.sp + head + row * p.pages.sr, sat = E4M3 ? page * p.pages.scale_sp + scale_head + row * p.pages.scale_sr : 0;
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            const int byte = 32 * c + 16 * h;  // (columns of 16 bits: 16 c + 8 h)
            const bool ok = there && byte < (E4M3 ? p.D : 2 * p.D);
            kr[c] = *static_cast<const u32x4*>(ok ? p.pages.k + at + byte : none);
            if constexpr (E4M3) ks[c] = *static_cast<const uint8_t*>(ok ? p.pages.ks + sat + c : none);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int y = lane + 64 * i, r = y / PC, c = y % PC, vkey = 32 * t + r, vrow = vkey - p.pages.page_of(vkey) * p.pages.size;
            const int vpage = __shfl(page, r);
            const bool ok = (uint32_t)vpage < (uint32_t)p.pages.pages && 16 * c < (E4M3 ? p.D : 2 * p.D);
            vr[i] = *static_cast<const u32x4*>(ok ? p.pages.v + vpage * p.pages.sp + head + vrow * p.pages.sr + 16 * c : none);
            if constexpr (E4M3)
                vs[i] = *static_cast<const uint8_t*>(ok ? p.pages.vs + vpage * p.pages.scale_sp + scale_head + vrow * p.pages.scale_sr + c / 2 : none);
        }
    };
    int t = part.first + wave, page = t < part.end ? look(t) : -1;
    if (t < part.end) load(t, page);
    if (t + WAVES < part.end) page = look(t + WAVES);
    SeqSums<HD> st;
    elem_t* V = region + wave * kRegion;
    const Tile<HD, false> tile(lane);
    for (; t < part.end; t += WAVES) {
        f32x16 s[1] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int y = lane + 64 * i;
            if constexpr (E4M3) {
                elem_t* to = V + (y / PC) * (HD + 8) + 16 * (y % PC);
                const float scale = scale_of(vs[i]);
                *reinterpret_cast<u32x4*>(to) = from_e4m3_8<T>(vr[i][0], vr[i][1], scale);
                *reinterpret_cast<u32x4*>(to + 8) = from_e4m3_8<T>(vr[i][2], vr[i][3], scale);
            } else {
                *reinterpret_cast<u32x4*>(V + (y / PC) * (HD + 8) + 8 * (y % PC)) = vr[i];
            }
        }
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            if constexpr (E4M3) {
                const float scale = scale_of(ks[c]);
                s[0] = Mma32<T>::run(from_e4m3_8<T>(kr[c][0], kr[c][1], scale), own[2 * c], s[0]);
                s[0] = Mma32<T>::run(from_e4m3_8<T>(kr[c][2], kr[c][3], scale), own[2 * c + 1], s[0]);
            } else {
                s[0] = Mma32<T>::run(kr[c], own[c], s[0]);
            }
        }
        if (t + WAVES < part.end) {
            load(t + WAVES, page);
            if (t + 2 * WAVES < part.end) page = look(t + 2 * WAVES);
        }
        if (32 * t + 32 <= whole) st.template take<false>(s, p.c, 0, h);
        else st.template take<true>(s, p.c, limit - 32 * t, h);
        wave_exchange();
        add_columns<T>(st.acc, tile, V, 0, s[0]);
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
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(out + 32 * dt + 8 * i) =
                f32x4{st.acc[dt][4 * i], st.acc[dt][4 * i + 1], st.acc[dt][4 * i + 2], st.acc[dt][4 * i + 3]};
    workgroup_barrier();
    for (int y = tid; y < rows * CH; y += 64 * WAVES) {
        const int row = y / CH, c8 = 8 * (y % CH);
        float top = -INFINITY, sum = 0.0f, o[8] = {};
#pragma unroll
        for (int k = 0; k < WAVES; ++k) top = fmaxf(top, stats[k * 32 + row]);
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            const float f = fast_exp2(stats[k * 32 + row] - ref);
            sum += f * stats[(WAVES + k) * 32 + row];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] += f * sums[(k * 32 + row) * kSum + c8 + j];
        }
        const SeqRow to(p, hk, r0 + row);
        if (p.splits > 1) {
            const int64_t place = seq_place(p, b, hk, r0 + row);
            if (split == 0 && c8 == 0) p.used[place] = part.used > 1 ? part.used : 0;
            if (part.used > 1) {
                const int64_t at = split * seq_places(p) + place;
                if (c8 == 0) p.stat[2 * at] = top, p.stat[2 * at + 1] = sum;
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    *reinterpret_cast<f32x4*>(p.part + at * HD + c8 + 4 * j) = f32x4{o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]};
                continue;
            }
        }
        const float f = sum == 0.0f || top == -INFINITY ? 0.0f : 1.0f / sum;
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = T::pack2(f == 0.0f ? 0.0f : o[2 * j] * f, f == 0.0f ? 0.0f : o[2 * j + 1] * f);
        store_chunk(p.o.head(0, to.hq) + (int64_t)(b.token + to.token) * p.o.sl, r, c8, p.D);
    }
}

// Joins the splits of seq_few: 16 threads to the columns of a row (eight each), `slices` of them to the splits, which meet in LDS.
template <typename T, int HD>
__global__ __launch_bounds__(kCtxThreads) void seq_join(SeqParams p) {
    __shared__ float met[kCtxThreads / 16][16][11];
    const int64_t all = seq_places(p), per = seq_group(p);
    const int slices = min(16, 1 << (32 - __builtin_clz(p.splits - 1))), group = threadIdx.x >> 4, slice = group % slices;
    const int64_t place = (int64_t)blockIdx.x * (16 / slices) + group / slices;
    const int c8 = 8 * (threadIdx.x & 15);
    int token = 0, hq = 0, used = 0;
    if (place < all) {
        const int64_t i = place % per;
        hq = (int)(place / per) * p.G;
        if (p.most == kSeqFew) {
            const int segment = (int)(i / kSeqFew), row = (int)(i % kSeqFew), first = seq_offset(p, segment);
            const int rows = max(0, seq_offset(p, segment + 1) - first) * p.G;
            if (row < rows && rows <= kSeqFew) used = p.used[place];
            token = first + row / p.G, hq += row % p.G;
        } else {
            // (rows of descending offsets belong to nobody, and the places of such are not written)
            token = (int)(i / p.G), hq += (int)(i % p.G);
            used = p.used[place];
        }
        used = min(used, p.splits);
    }
    const bool some = used > 0 && c8 < HD;
    float top = -INFINITY, sum = 0.0f, y[8] = {};
    const auto add = [&](float other_top, float other_sum, const float* other) {
        const float now = fmaxf(top, other_top), ref = now == -INFINITY ? 0.0f : now, f = fast_exp2(top - ref), g = fast_exp2(other_top - ref);
        top = now;
        sum = f * sum + g * other_sum;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = f * y[j] + g * other[j];
    };
    if (some) {
        for (int s = slice; s < used; s += slices) {
            const int64_t at = s * all + place;
            const f32x4 a = *reinterpret_cast<const f32x4*>(p.part + at * HD + c8), c = *reinterpret_cast<const f32x4*>(p.part + at * HD + c8 + 4);
            const float other[8] = {a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
            add(p.stat[2 * at], p.stat[2 * at + 1], other);
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
    const float f = sum == 0.0f || top == -INFINITY ? 0.0f : 1.0f / sum;
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = T::pack2(f == 0.0f ? 0.0f : y[2 * j] * f, f == 0.0f ? 0.0f : y[2 * j + 1] * f);
    store_chunk(p.o.head(0, hq) + (int64_t)token * p.o.sl, o, c8, p.D);
}

}  // namespace sjvp
