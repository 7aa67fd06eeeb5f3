// Forward kernels of the attention over packed sequences and over a paged cache (sjvp_seq.hpp).
#pragma once
#include "sjvp_seq.hpp"
#include "sjvp_w16.hpp"

namespace sjvp {

// The rows of a block: those of all heads that share a key head, token by token (row = token * G + head of the group), so that they read their
// keys once and a short sequence fills a block.
struct SeqRow {
    int token, hq;  // token within the segment
    __device__ __forceinline__ SeqRow(const SeqParams& p, int hk, int row) : token(row / p.G), hq(hk * p.G + row % p.G) {}
};

// Splits of the tiles of a sequence's keys: of split_tiles or more, as many as the launch has at most.
struct SeqSplit {
    int used, first, end;
    __device__ __forceinline__ SeqSplit(const SeqParams& p, int tiles, int split) {
        const int per = max(p.split_tiles, (tiles + p.splits - 1) / p.splits);
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

// Many rows: four waves of 32 rows share tiles of 64 keys, two tiles of K and V in LDS, one barrier to a tile.  Scores are transposed (32x32x16), so that a
// row is a lane pair, its maximum and sum need one exchange, and P goes into the second contraction from registers.  Tiles that every row
// sees as a whole have a loop without masks.
//
// Bound by the matrix unit and the exponentials alike: two prompts of 4915 and 8192 tokens, Hq=16 Hkv=2 D=128, causal, 346 us = 1.09 PFLOP/s (a
// 16384^3 product: 1.36), the matrix unit busy 59 % and the vector unit 58 %; 64 sequences of 16 to 128 tokens, 12 heads, D=64, whole, 12.5 us =
// 2.3 TB/s, where a workgroup is one or two tiles and its start and end.  On pages (eight prompts of 128 to 512 tokens on 2048 to 8192, Hq=16
// Hkv=4 D=128 e4m3) 166 us and 20 for the join, 0.64 PFLOP/s: a tile of 8-bit numbers goes through registers, with 10 vector instructions to a matrix
// instruction in place of 7; 16-bit pages, by LDS-DMA, take 171 us in place of 180 with the join: with two waves to a SIMD a wave's contractions, exponentials and waits for the next
// tile stand one behind the other for the most part.
template <typename T, int HD, bool PAGED, typename FEED>
__global__ __launch_bounds__(kCtxThreads, HD <= 64 ? 4 : 2) void seq_fwd(SeqParams p) {
    if constexpr (FEED::kDma) __builtin_assume(p.D % 8 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kTile = SeqTile<HD>::kElems;
    constexpr bool kAhead = !PAGED && FEED::kDma && HD == 128;
    elem_t* tiles = reinterpret_cast<elem_t*>(smem);  // K [2], V [2]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % p.Hkv, x = blockIdx.x / p.Hkv, split = PAGED ? x / p.slots : 0;
    const SeqBlock b = PAGED ? seq_block_most_keys_first<kCtxOwned, kCtxTile>(p, x - split * p.slots, lane)
                             : seq_block_long_first<kCtxOwned>(p, x, p.G, false, lane);
    const int all = b.tokens * p.G;
    if (!b.some || all < p.least || all > p.most) return;
    const SeqKeys<PAGED> keys(p, b);
    const int r0 = b.row0 + 32 * wave, rows = min(max(all - r0, 0), 32);
    const SeqRow mine(p, hk, min(r0 + (lane & 31), all - 1));
    const bool ok = (lane & 31) < rows;
    const int limit = keys.seen(p, mine.token);
    const int n = keys.seen(p, (min(b.row0 + kCtxOwned, all) - 1) / p.G), whole = keys.seen(p, b.row0 / p.G);  // keys of the last, the first row
    const int n_wave = rows > 0 ? keys.seen(p, (r0 + rows - 1) / p.G) : 0;

    const SeqSplit part(p, (n + kCtxTile - 1) / kCtxTile, split);
    if (PAGED && split >= part.used) return;
    u32x4 own[HD / 16];
    own_operands<HD>(own, p.q.head(0, mine.hq) + (int64_t)(b.token + mine.token) * p.q.sl, ok, h, p.D);
    const int t0 = PAGED ? part.first : 0, nt = PAGED ? part.end : (n + kCtxTile - 1) / kCtxTile;
    FEED feed(p, b, hk, tid);
    SeqTile<HD> at(tiles, lane);
    SeqSums<HD> st;
    constexpr int kHalf = 32 * SeqTile<HD>::kLd * 2, kV = 2 * SeqTile<HD>::kBytes;
    int step = SeqTile<HD>::kBytes;
    const auto k_place = [&](int t) { return tiles + ((t - t0) & 1) * kTile; };
    const auto v_place = [&](int t) { return tiles + (2 + ((t - t0) & 1)) * kTile; };
    // tile t's values that are not finite  (written out here: through the functions that the backward calls, which do the same, the compiler places
    // the loops so that two prompts of 5000 and 8192 tokens, Hq=16 Hkv=2 D=128, take 355 us in place of 346)
    const auto care = [&](int t) {
        elem_t* V = v_place(t);
        bool some = false;
        for (int x = tid; x < kTile / 8; x += kCtxThreads) {
            const int row = x / SeqTile<HD>::PP, c = x % SeqTile<HD>::PP ^ SeqTile<HD>::swz(row);
            if (HD == SeqTile<HD>::kLd || 8 * c < HD) some = some || any_not_finite<T>(reinterpret_cast<const u32x4*>(V)[x]);  // (not what pads a row)
        }
        if (!workgroup_barrier_or(some)) return;
        for (int j = 0; j < min(limit - t * kCtxTile, kCtxTile); ++j) {
            const elem_t* from = V + j * SeqTile<HD>::kLd + 4 * h;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                const f32x4 more = only_not_finite<T>(from + 8 * (c ^ SeqTile<HD>::swz(j)));
#pragma unroll
                for (int i = 0; i < 4; ++i) st.acc[c / 4][4 * (c % 4) + i] += more[i];
            }
        }
        workgroup_barrier();
        for (int x = tid; x < kTile / 8; x += kCtxThreads) {
            u32x4* piece = reinterpret_cast<u32x4*>(V) + x;
            *piece = only_finite<T>(*piece);
        }
        workgroup_barrier();
    };
    // the tiles that all rows see as a whole have a loop without masks
    const int free = max(min(whole / kCtxTile, nt), t0);
    const auto walk = [&](auto&& tile) {
        int t = t0;
        for (; t < free; ++t) tile(t, std::false_type{});
        for (; t < nt; ++t) tile(t, std::true_type{});
    };
    if constexpr (kAhead) {
        // K runs a tile ahead of V, so that the scores of the next tile are made beside the exponentials of this one.
        if (nt) {
            feed.request_k(p, 0, n, k_place(0), wave);
            feed.request_v(p, 0, n, v_place(0), wave);
            if (nt > 1) feed.request_k(p, 1, n, k_place(1), wave);
        }
        feed.arrived();
        workgroup_barrier();
        f32x16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = at.template scores<T>(u * kHalf, own);
        workgroup_barrier();
        walk([&](int t, auto masked) {
            if (t + 1 < nt) feed.request_v(p, t + 1, n, v_place(t + 1), wave);
            if (t + 2 < nt) feed.request_k(p, t + 2, n, k_place(t), wave);
            if (decltype(masked)::value && p.causal) care(t);
            at.move(step);
            if (t * kCtxTile < n_wave) {
                st.template raise<decltype(masked)::value>(s, p.c, limit - t * kCtxTile, h);
                f32x16 next[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) next[u] = at.template scores<T>(u * kHalf, own);
                st.exponentials(s, p.c);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    at.template add_columns<T>(st.acc, kV - step + u * kHalf, s[u]);
                    s[u] = next[u];
                }
            }
            step = -step;
            feed.arrived();
            workgroup_barrier();
        });
    } else {
        if (t0 < nt) {
            feed.look(p, t0, n);
            feed.request(p, t0, n, k_place(t0), v_place(t0), wave);
            if (t0 + 1 < nt) feed.look(p, t0 + 1, n);
            feed.deliver(p, k_place(t0), v_place(t0), tid);
        }
        feed.arrived();
        workgroup_barrier();
        walk([&](int t, auto masked) {
            const bool more = t + 1 < nt;
            if (more) {
                feed.request(p, t + 1, n, k_place(t + 1), v_place(t + 1), wave);
                if (t + 2 < nt) feed.look(p, t + 2, n);
            }
            if (decltype(masked)::value && p.causal) care(t);
            if (t * kCtxTile < n_wave) {
                // (the second half's scores beside the first half's exponentials, at D in 65 to 96 alone: four sequences of 1024 to 2048 tokens, Hq=16 Hkv=4
                // D=96 50.4 us in place of 53.9; eight of D=64, whole, 109.6 in place of 108.1; chunks on pages at D=96 71.0 in place of 70.6)
                constexpr int kParts = !PAGED && HD == 96 ? 2 : 1;
                f32x16 s[kParts][2 / kParts];
#pragma unroll
                for (int u = 0; u < 2; ++u) s[u * kParts / 2][u % (2 / kParts)] = at.template scores<T>(u * kHalf, own);
#pragma unroll
                for (int i = 0; i < kParts; ++i) {
                    st.template take<decltype(masked)::value>(s[i], p.c, limit - t * kCtxTile - 32 * i, h);
#pragma unroll
                    for (int j = 0; j < 2 / kParts; ++j) at.template add_columns<T>(st.acc, kV + (i + j) * kHalf, s[i][j]);
                }
            }
            at.move(step);
            step = -step;
            if (more) feed.deliver(p, k_place(t + 1), v_place(t + 1), tid);
            feed.arrived();
            workgroup_barrier();
        });
    }
    const float both = halves_sum(st.l), l = limit > 0 ? both : 0.0f, f = l == 0.0f ? 0.0f : 1.0f / l;
    if (p.lse && h == 0 && ok)
        *reinterpret_cast<f32x2*>(p.lse + 2 * ((int64_t)mine.hq * p.T + b.token + mine.token)) = f32x2{l == 0.0f ? 0.0f : st.ref, l};
    if constexpr (PAGED) {
        if (p.splits > 1 && ok) {
            const int64_t place = seq_place(p, b, hk, r0 + (lane & 31));
            if (split == 0 && h == 0) p.used[place] = part.used > 1 ? part.used : 0;
            if (part.used > 1) {
                const int64_t at = split * seq_places(p) + place;
                if (h == 0) p.stat[2 * at] = st.m == -INFINITY ? -INFINITY : st.ref, p.stat[2 * at + 1] = both;
                float* out = p.part + at * HD + 4 * h;
#pragma unroll
                for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<f32x4*>(out + 32 * dt + 8 * i) =
                            f32x4{st.acc[dt][4 * i], st.acc[dt][4 * i + 1], st.acc[dt][4 * i + 2], st.acc[dt][4 * i + 3]};
            }
        }
        if (part.used > 1) return;
    }
    store_rows_at<T, HD>(st.acc, f, rows, tiles + wave * 32 * (HD + 8), lane, p.D, [&](int row) {
        const SeqRow to(p, hk, r0 + row);
        return p.o.head(0, to.hq) + (int64_t)(b.token + to.token) * p.o.sl;
    });
}

// Maximum and sum over the four lanes (l, l ^ 16, l ^ 32, l ^ 48) of a row.
__device__ __forceinline__ float quarters_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Few rows: 16 or 32 rows to a block (NC sets of 16) and waves that share out its keys: each runs over tiles of 32 keys of its own, K straight from
// memory into the operand's registers, V through a region of LDS that no other wave reads, so that nothing but the end is synchronised.  The
// sums of the waves are joined in LDS; with several splits of the keys they go to memory for seq_join.
//
// The matrix instructions are 16x16x32 (tile algebra in sjvp_w16.hpp), so that a step of a group of heads, some four to sixteen rows, leaves
// little of them idle, and with one set of rows a wave needs 128 registers (16-bit numbers above D = 96: 162): four (three) waves to a SIMD hold
// twice as many loads in flight as the 32-wide form did.
//
// Bound by memory where sequences are many (a token each of 64 sequences of 2048 to 8192, Hq=16 Hkv=4 D=128 e4m3: 75 us = 4.6 TB/s, a copy makes
// 5.2), by the latency of offsets, tables and two tiles one behind the other where they are few (four tokens on 29491 and 32769, Hq=16 Hkv=2, 16 bits: 20 us,
// 3.2 TB/s; a token on 128: 5 us).
// E4M3: the cache's numbers have 8 bits; a lane's 16 bytes are columns of two chunks of 32 then, and q is read in that order.
template <typename T, int HD, bool E4M3, int NC, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NC == 1 ? (E4M3 || HD <= 96 ? 4 : 3) : HD <= 64 ? 4 : 2) void seq_few(SeqParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int R = 16 * NC, kLd = HD + 8, kSum = HD + 4, CH = HD / 8, KC = HD / 32, DT = HD / 16;
    elem_t* region = reinterpret_cast<elem_t*>(smem);  // [WAVES][32] rows of V, then the waves' sums [WAVES][R][HD + 4] fp32
    float* sums = reinterpret_cast<float*>(smem);
    float* stats = sums + WAVES * R * kSum;  // [WAVES][R] maximum, then sum
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), y = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % p.Hkv, x = blockIdx.x / p.Hkv, slot = x % p.slots, split = x / p.slots;
    const SeqBlock b = p.most == kSeqFew ? seq_block_few<R>(p, slot) : seq_block<R, true>(p, slot, p.G, lane);
    const int all = b.tokens * p.G;
    if (!b.some || all > p.most) return;
    const SeqKeys<true> keys(p, b);
    const int r0 = b.row0, rows = min(all - r0, R);
    const int n = keys.seen(p, (r0 + rows - 1) / p.G), whole = keys.seen(p, r0 / p.G);
    const SeqSplit part(p, (n + 31) / 32, split);
    if (split >= part.used) return;

    // column of the eight numbers that step c of a contraction over the head dimension has in this lane
    const auto column = [&](int c) { return !E4M3 || (KC % 2 && c == KC - 1) ? 32 * c + 8 * g : 64 * (c / 2) + 16 * g + 8 * (c % 2); };
    u32x4 own[NC][KC];
    int limit[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const SeqRow mine(p, hk, min(r0 + 16 * i + y, all - 1));
        limit[i] = keys.seen(p, mine.token);
        const elem_t* q = p.q.head(0, mine.hq) + (int64_t)(b.token + mine.token) * p.q.sl;
#pragma unroll
        for (int c = 0; c < KC; ++c) own[i][c] = 16 * i + y < rows ? load_chunk(q, column(c), p.D) : u32x4{0u, 0u, 0u, 0u};
    }
    // K and V of the rows 16 u + lane % 16 of a tile: pieces of 16 bytes, the last one of an odd number of 8-bit chunks of 8
    constexpr int NP = E4M3 ? (KC + 1) / 2 : KC;
    u32x4 kr[2][NP], vr[2][NP];
    uint32_t ks[2] = {}, vs[2] = {};
    const int* table = p.pages.table + (b.segment - 1) * p.pages.table_stride;
    const unsigned char *kp = p.pages.k + hk * p.pages.sh, *vp = p.pages.v + hk * p.pages.sh;
    const unsigned char *ksp = p.pages.ks + hk * p.pages.scale_sh, *vsp = p.pages.vs + hk * p.pages.scale_sh;
    const void* none = &kZeroPiece;
    int page[2];
    const auto look = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int key = 32 * t + 16 * u + y;
            page[u] = key < n ? table[p.pages.page_of(key)] : -1;
        }
    };
    const auto load = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int key = 32 * t + 16 * u + y, row = key - p.pages.page_of(key) * p.pages.size;
            const bool there = (uint32_t)page[u] < (uint32_t)p.pages.pages;
            const int64_t at = p.pages.at(page[u], row);
#pragma unroll
            for (int c = 0; c < NP; ++c) {
                if (E4M3 && KC % 2 && c == NP - 1) {
                    const int byte = 32 * (KC - 1) + 8 * g;
                    const bool ok = there && byte < p.D;
                    const u32x2 a = global<u32x2>(ok ? kp + at + byte : none), d = global<u32x2>(ok ? vp + at + byte : none);
                    kr[u][c] = u32x4{a[0], a[1], 0u, 0u}, vr[u][c] = u32x4{d[0], d[1], 0u, 0u};
                } else {
                    const int byte = 64 * c + 16 * g;
                    const bool ok = there && byte < (E4M3 ? p.D : 2 * p.D);
                    kr[u][c] = global<u32x4>(ok ? kp + at + byte : none);
                    vr[u][c] = global<u32x4>(ok ? vp + at + byte : none);
                }
            }
            if constexpr (E4M3) {
                const int64_t sat = p.pages.scale_at(page[u], row);
                ks[u] = scale_codes<KC>(there ? ksp + sat : none, p.pages.scale_words);
                vs[u] = scale_codes<KC>(there ? vsp + sat : none, p.pages.scale_words);
            }
        }
    };
    // step c's eight numbers of a row, from its pieces
    const auto operand = [&](const u32x4* r, uint32_t codes, int c) {
        if constexpr (!E4M3) return r[c];
        if (KC % 2 && c == KC - 1) return from_e4m3_8<T>(r[c / 2][0], r[c / 2][1], scale_of(codes >> (8 * c) & 0xffu));
        // columns 64 (c / 2) + 16 g ..: the first or the second group of 32 of the pair
        return from_e4m3_8<T>(r[c / 2][2 * (c % 2)], r[c / 2][2 * (c % 2) + 1], scale_of(codes >> (16 * (c / 2) + 8 * (g >> 1)) & 0xffu));
    };
    int t = part.first + wave;
    if (t < part.end) {
        look(t);
        load(t);
    }
    if (t + WAVES < part.end) look(t + WAVES);
    f32x4 acc[NC][DT] = {};
    float m[NC], ref[NC], l[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) m[i] = -INFINITY, ref[i] = 0.0f, l[i] = 0.0f;
    elem_t* V = region + wave * 32 * kLd;
    // transposing reads: lane 4j + i of 16 supplies row 4g + j, columns 4i .. 4i+3, lane i receives column i
    const elem_t* tr = V + (4 * g + (y >> 2)) * kLd + 4 * (y & 3);
    for (; t < part.end; t += WAVES) {
        f32x4 s[NC][2] = {};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                *reinterpret_cast<u32x4*>(V + (16 * u + y) * kLd + column(c)) = operand(vr[u], vs[u], c);
                const u32x4 k = operand(kr[u], ks[u], c);
#pragma unroll
                for (int i = 0; i < NC; ++i) s[i][u] = T::mfma16(k, own[i][c], s[i][u]);
            }
        if (t + WAVES < part.end) {
            load(t + WAVES);
            if (t + 2 * WAVES < part.end) look(t + 2 * WAVES);
        }
        const bool masked = 32 * t + 32 > whole;
        if (masked && whole < n) {
            wave_exchange();
            bool some = false;
            for (int x = lane; x < 32 * CH; x += 64) some = some || any_not_finite<T>(*reinterpret_cast<const u32x4*>(V + x / CH * kLd + 8 * (x % CH)));
            if (__builtin_amdgcn_ballot_w64(some)) {
                for (int j = 0; j < 32; ++j)
#pragma unroll
                    for (int i = 0; i < NC; ++i)
                        if (32 * t + j < limit[i])
#pragma unroll
                            for (int d = 0; d < DT; ++d) acc[i][d] += only_not_finite<T>(V + j * kLd + 16 * d + 4 * g);
                wave_exchange();
                for (int x = lane; x < 32 * CH; x += 64) {
                    u32x4* piece = reinterpret_cast<u32x4*>(V + x / CH * kLd + 8 * (x % CH));
                    *piece = only_finite<T>(*piece);
                }
            }
        }
        u32x4 pr[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (masked) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (32 * t + 16 * u + 4 * g + j >= limit[i]) s[i][u][j] = -INFINITY;
            }
            float top = s[i][0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top = fmaxf(top, s[i][j >> 2][j & 3]);
            top *= p.c;
            if (__builtin_amdgcn_ballot_w64(top > m[i] + 8.0f)) {
                const float grown = fmaxf(m[i], quarters_max(top)), now = grown == -INFINITY ? 0.0f : grown;
                const float f = m[i] == -INFINITY ? 1.0f : fast_exp2(ref[i] - now);
                m[i] = grown, ref[i] = now;
                l[i] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[i][d] *= f;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][u][j] = fast_exp2(__builtin_fmaf(s[i][u][j], p.c, -ref[i]));
                    l[i] += s[i][u][j];
                }
            pr[i] = pack_b16<T>(s[i][0], s[i][1]);
        }
        wave_exchange();
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tr + 16 * d)));
            const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tr + 16 * kLd + 16 * d)));
            const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
            for (int i = 0; i < NC; ++i) acc[i][d] = T::mfma16(v, pr[i], acc[i][d]);
        }
        wave_exchange();
    }
    workgroup_barrier();  // the sums take the place of the V tiles
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const float sum = quarters_sum(l[i]);
        if (g == 0) {
            stats[wave * R + 16 * i + y] = m[i] == -INFINITY ? -INFINITY : ref[i];
            stats[(WAVES + wave) * R + 16 * i + y] = sum;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(sums + (wave * R + 16 * i + y) * kSum + 16 * d + 4 * g) = acc[i][d];
    }
    workgroup_barrier();
    for (int z = tid; z < rows * CH; z += 64 * WAVES) {
        const int row = z / CH, c8 = 8 * (z % CH);
        float top = -INFINITY, sum = 0.0f, o[8] = {};
#pragma unroll
        for (int k = 0; k < WAVES; ++k) top = fmaxf(top, stats[k * R + row]);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            const float f = fast_exp2(stats[k * R + row] - base);
            sum += f * stats[(WAVES + k) * R + row];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] += f * sums[(k * R + row) * kSum + c8 + j];
        }
        const SeqRow to(p, hk, r0 + row);
        if (p.used_many && split == 0 && c8 == 0) p.used_many[hk * (int64_t)p.T * p.G + (int64_t)b.token * p.G + r0 + row] = 0;
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
        // (a row that sees nothing sums to exactly zero; scores that are all NaN have no maximum either)
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = T::pack2(f == 0.0f ? 0.0f : o[2 * j] * f, f == 0.0f ? 0.0f : o[2 * j + 1] * f);
        store_chunk(p.o.head(0, to.hq) + (int64_t)(b.token + to.token) * p.o.sl, r, c8, p.D);
    }
}

// Joins the splits of seq_few or seq_fwd: 16 threads to the columns of a row (eight each), `slices` of them to the splits, which meet in LDS.  A launch of
// its own, 4 to 7 us for few rows, whose least is 4: a join by the last workgroup would need counters that start at zero, which is a launch
// too.  41000 rows of 128 in one to four splits, some 60 MB of sums: 19 us = 3.7 TB/s.
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
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = T::pack2(f == 0.0f ? 0.0f : y[2 * j] * f, f == 0.0f ? 0.0f : y[2 * j + 1] * f);
    store_chunk(p.o.head(0, hq) + (int64_t)token * p.o.sl, o, c8, p.D);
}

}  // namespace sjvp
