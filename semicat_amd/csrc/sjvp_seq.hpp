// Attention over packed sequences and over a paged cache: parameters and device building blocks (kernels: sjvp_seq_fwd.hpp,
// sjvp_seq_bwd.hpp, sjvp_paged.hip; tile algebra: sjvp_ctx.hpp).
//
//   s[i][j] = scale q_i.k_j    for the keys j of the query's own sequence, causal: up to its own position
//   p = softmax over j,  o_i = sum_j p[i][j] v_j
//
// Sequences stand one behind the other in tensors of T rows; offsets [B+1] say where.  The rows in front of the first one and behind
// the last one are two more segments, without keys, so that every row of a result is written by the same code: segment 0 is
// [0, offsets[0]), segment x in 1 .. B is sequence x - 1, segment B + 1 ends at T.  Offsets are clamped to T; what is not ascending
// gives rows of no use, none out of bounds.
//
// Which segment a workgroup serves is found on the device, so that the host reads no lengths: blocks of R rows of a segment take the slots
//   floor(offset / R) + segment, ...
// which never meet, since floor(a / R) + ceil(n / R) <= floor((a + n) / R) + 1; the slot of a workgroup gives its segment by a search of 64
// places at a time.  T / R + B + 2 slots hold all blocks, at most B + 2 of them idle.
#pragma once
#include "sjvp_ctx.hpp"

namespace sjvp {

// Pages of a cache: [pages, heads, size, D] numbers of 16 or 8 bits, the latter with a power of two for each 32 columns (8-bit exponents
// [pages, heads, size, ceil(D / 32)]).  Strides in bytes, the same of K and V.  Position x of sequence b stands in row x % size of page
// table[b][x / size]; a page number that the cache has not reads as zeros.
struct SeqPages {
    unsigned char *k, *v, *ks, *vs;
    int64_t sh, scale_sh;
    uint32_t sp, sr, scale_sp, scale_sr;  // (of 32 bits: an instruction to a product in place of four; 79 sequences of up to 11 tokens on 1280 to
                                          // 5120, 16 heads of 32, e4m3: 62 us in place of 70)
    const int* table;
    int64_t table_stride;
    int pages, size, capacity;  // capacity: positions that a row of the table has
    int scale_words;            // the exponents of a row are one word of memory (32 or 16 bits)
    uint32_t magic, shift;      // x / size = mulhi(2 x, magic) >> shift below 2^30
    __device__ __forceinline__ int64_t at(int page, int row) const { return (int64_t)((uint64_t)(uint32_t)page * sp + (uint64_t)(uint32_t)row * sr); }
    __device__ __forceinline__ int64_t scale_at(int page, int row) const {
        return (int64_t)((uint64_t)(uint32_t)page * scale_sp + (uint64_t)(uint32_t)row * scale_sr);
    }
    __device__ __forceinline__ int page_of(int x) const { return (int)(__umulhi(2u * (uint32_t)x, magic) >> shift); }
};

// Rows of a sequence that seq_few serves beside seq_fwd (48 sequences of 0 to 80 tokens on up to 2048, Hq=16 Hkv=4 D=128: 68 us; with 64 74, 128 85).
constexpr int kSeqFew = 32;

struct SeqParams {
    CtxView q, k, v, o, g, dq, dk, dv;  // [T,H,D], sb unused
    float *lse, *folded;                // [Hq,T][2]: (m, l) of each row; [3][Hq,T]: row_stat_folded, -delta
    float *part, *stat;                 // sums of split work: [splits][seq_places] of HD floats, and their (maximum, sum)
    int *used, *used_many;              // splits that a row's sums stand in (0: in none); seq_few beside a split seq_fwd: those of seq_fwd
    const int *offsets, *lengths;       // offsets null: one row each
    int B, T, Hq, Hkv, G, D, causal;
    float scale, c;                     // c = scale * log2(e)
    int slots, splits, split_tiles;     // split_tiles: tiles (of 32 keys, seq_fwd: of 64) that a split has at least
    int least, most;                    // query rows (of all heads of a group) of the sequences that a launch serves
    SeqPages pages;
};

__device__ __forceinline__ int seq_offset(const SeqParams& p, int x) {
    if (x == 0) return 0;
    if (x >= p.B + 2) return p.T;
    return min(max(p.offsets ? p.offsets[x - 1] : x - 1, 0), p.T);
}

// The block of R rows (of `heads` rows to a token) that a workgroup serves, and the length that the cache has of its sequence.  In the last step of the
// search the lanes hold the offsets and lengths of neighbouring segments, so that a workgroup waits for memory once (up to 62 sequences) before it
// knows its rows and keys.
struct SeqBlock {
    int segment, token, tokens, row0;  // first token and number of tokens of the segment; first row of the block within it
    int held;
    bool some;
};
template <int R, bool PAGED = false>
__device__ __forceinline__ SeqBlock seq_block(const SeqParams& p, int slot, int heads, int lane) {
    int lo = 0, hi = p.B + 2;  // the segment lies in [lo, hi)
    while (hi - lo > 64) {
        const int step = (hi - lo + 63) / 64, x = lo + lane * step;
        const bool there = x < hi && seq_offset(p, x) * heads / R + x <= slot;
        const int n = __popcll(__builtin_amdgcn_ballot_w64(there || lane == 0));
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    const int x = lo + lane, at = seq_offset(p, x), next = seq_offset(p, x + 1);
    const int held = PAGED && x >= 1 && x <= p.B ? p.lengths[x - 1] : 0;
    const int mine = __popcll(__builtin_amdgcn_ballot_w64(lane == 0 || (x < hi && at * heads / R + x <= slot))) - 1;
    SeqBlock b;
    b.segment = __builtin_amdgcn_readfirstlane(lo + mine);
    b.token = __builtin_amdgcn_readlane(at, mine);
    b.tokens = max(0, __builtin_amdgcn_readlane(next, mine) - b.token);
    b.held = __builtin_amdgcn_readlane(held, mine);
    b.row0 = (slot - (b.token * heads / R + b.segment)) * R;
    b.some = b.row0 >= 0 && b.row0 < b.tokens * heads;  // (descending offsets may lead to a segment that begins behind the slot)
    return b;
}

// Beside a launch that serves the longer sequences, kSeqFew / R slots to a segment.
template <int R>
__device__ __forceinline__ SeqBlock seq_block_few(const SeqParams& p, int slot) {
    SeqBlock b;
    b.segment = slot / (kSeqFew / R), b.row0 = slot % (kSeqFew / R) * R;
    b.token = seq_offset(p, b.segment), b.tokens = max(0, seq_offset(p, b.segment + 1) - b.token);
    b.held = b.segment >= 1 && b.segment <= p.B ? p.lengths[b.segment - 1] : 0;
    b.some = b.row0 < b.tokens * p.G;
    return b;
}

__device__ __forceinline__ int lanes_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false);  // turned by 8, 4, 2, 1 of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false);
    return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) + __builtin_amdgcn_readlane(x, 48);
}

// The same for causal launches, whose blocks take the longer the further they are from the front of their sequence (or, with `back`, from its
// end): the rank-th block in descending order of that distance, over all sequences, so that the launch does not end with long ones.  With up to 62
// sequences; with more the plain order does.  C(j) blocks have a distance of j or more; j with C(j) > rank >= C(j + 1) is the block's.
template <int R>
__device__ __forceinline__ SeqBlock seq_block_long_first(const SeqParams& p, int rank, int heads, bool back, int lane) {
    if (!p.causal) return seq_block<R>(p, rank, heads, lane);
    if (p.B + 2 > 64) return seq_block<R>(p, back ? rank : p.slots - 1 - rank, heads, lane);
    const int at = seq_offset(p, min(lane, p.B + 2)), tokens = lane < p.B + 2 ? max(0, seq_offset(p, lane + 1) - at) : 0;
    const int blocks = (tokens * heads + R - 1) / R;
    int lo = 0, hi = 1;
    while (__builtin_amdgcn_ballot_w64(blocks > hi)) hi *= 2;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (lanes_sum(max(0, blocks - mid)) > rank) lo = mid;
        else hi = mid;
    }
    const int left = rank - lanes_sum(max(0, blocks - lo - 1));
    const uint64_t those = __builtin_amdgcn_ballot_w64(blocks > lo);
    const uint64_t one = __builtin_amdgcn_ballot_w64(blocks > lo && __popcll(those & ((uint64_t(1) << lane) - 1)) == left);
    SeqBlock b;
    b.some = one != 0;
    b.segment = one ? __builtin_ctzll(one) : 0;
    b.token = __builtin_amdgcn_readlane(at, b.segment);
    b.tokens = __builtin_amdgcn_readlane(tokens, b.segment);
    b.row0 = (back ? __builtin_amdgcn_readlane(blocks, b.segment) - 1 - lo : lo) * R;
    b.held = 0;
    return b;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int lanes_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // from 1, 2, 4, 8 lanes below in a row of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the last lane of a row to the next row
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // that of the first half to the second one
    return x;
}

// The blocks of the paged attention in descending order of their sequences' keys (in 16 classes), for the same reason, over the sequences that the
// launch serves; a sequence's last block first.
template <int R, int TILE>
__device__ __forceinline__ SeqBlock seq_block_most_keys_first(const SeqParams& p, int rank, int lane) {
    if (p.B + 2 > 64) return seq_block<R, true>(p, p.slots - 1 - rank, p.G, lane);
    const int at = seq_offset(p, min(lane, p.B + 2)), tokens = lane < p.B + 2 ? max(0, seq_offset(p, lane + 1) - at) : 0;
    const int held = lane >= 1 && lane <= p.B ? p.lengths[lane - 1] : 0, rows = tokens * p.G;
    const int blocks = rows >= p.least && rows <= p.most ? (rows + R - 1) / R : 0;
    int key = min(max(held, 0), p.pages.capacity) / TILE;
    while (__builtin_amdgcn_ballot_w64(key > 15)) key >>= 1;
    int lo = 0, hi = 16;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (lanes_sum(key >= mid ? blocks : 0) > rank) lo = mid;
        else hi = mid;
    }
    const int left = rank - lanes_sum(key > lo ? blocks : 0), upto = lanes_scan(key == lo ? blocks : 0);
    const uint64_t those = __builtin_amdgcn_ballot_w64(upto > left);
    SeqBlock b;
    b.some = those != 0;
    b.segment = those ? __builtin_ctzll(those) : 0;
    b.token = __builtin_amdgcn_readlane(at, b.segment);
    b.tokens = __builtin_amdgcn_readlane(tokens, b.segment);
    b.held = __builtin_amdgcn_readlane(held, b.segment);
    b.row0 = (__builtin_amdgcn_readlane(upto, b.segment) - 1 - left) * R;
    return b;
}

// Keys of a segment and the position of its first query among them.
template <bool PAGED>
struct SeqKeys {
    int keys, start;
    __device__ __forceinline__ SeqKeys(const SeqParams& p, const SeqBlock& b) {
        const bool sequence = b.segment >= 1 && b.segment <= p.B;
        if constexpr (PAGED) {
            const int length = sequence ? max(b.held, 0) : 0;
            keys = min(length, p.pages.capacity);
            start = length - b.tokens;  // (a length beyond the table: the positions that the table has not hold no keys)
        } else {
            keys = sequence ? b.tokens : 0;
            start = 0;
        }
    }
    // keys that query i sees
    __device__ __forceinline__ int seen(const SeqParams& p, int i) const { return p.causal ? max(0, min(keys, start + i + 1)) : keys; }
};

// Two 8-bit numbers of a word, times a power of two, as two 16-bit ones.
template <typename T>
__device__ __forceinline__ uint32_t from_e4m3(uint32_t word, float scale, bool high) {
    if constexpr (std::is_same_v<T, Bf16>) {
        return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true))
                    : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false));
    } else {
        return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, true))
                    : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, false));
    }
}
template <typename T>
__device__ __forceinline__ u32x4 from_e4m3_8(uint32_t a, uint32_t b, float scale) {
    return u32x4{from_e4m3<T>(a, scale, false), from_e4m3<T>(a, scale, true), from_e4m3<T>(b, scale, false), from_e4m3<T>(b, scale, true)};
}
// 2^(code - 127)
__device__ __forceinline__ float scale_of(uint32_t code) { return __uint_as_float(code << 23); }

// 16 bytes of zeros, for the lanes of a copy that have no row.
static __device__ const u32x4 kZeroPiece = {0u, 0u, 0u, 0u};

// A load from memory.  (Of a pointer that is one of two, the compiler does not know that neither points to LDS; the loads that it makes then count as LDS
// reads too, so that every wait for LDS waits for them: B=2 Hq=16 Hkv=2 four tokens on 32769 D=128 32 us.)
template <typename V>
__device__ __forceinline__ V global(const void* at) {
    return *(const __attribute__((address_space(1))) V*)(uintptr_t)at;
}

// The exponent codes of a row, a byte to each 32 columns.
template <int GROUPS>
__device__ __forceinline__ uint32_t scale_codes(const void* at, bool words) {
    if constexpr (GROUPS == 4)
        if (words) return global<uint32_t>(at);
    if constexpr (GROUPS == 2)
        if (words) return global<uint16_t>(at);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) codes |= (uint32_t)global<uint8_t>(static_cast<const uint8_t*>(at) + i) << (8 * i);
    return codes;
}

// Orders the instructions of a stretch without branches: LDS reads run `AHEAD` groups of READS ahead of the STEPS groups of MFMAS matrix
// instructions that use them.  (Left to itself the compiler puts a read right in front of its use where registers are short, and every matrix
// instruction waits for LDS.)
template <int STEPS, int READS, int MFMAS, int AHEAD>
__device__ __forceinline__ void reads_ahead() {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
    for (int i = 0; i < STEPS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, MFMAS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) __builtin_amdgcn_sched_group_barrier(0x008, MFMAS, 0);
}

// Infinities and NaN in rows that a causal query (or key) does not see: a contraction makes NaN of them by a probability of zero, for every query
// of the tile.  Tiles that some queries see in part are looked at before they are used; such numbers are added one by one to what sees
// them, and taken out of the tile.  The backward finds them in the scores, the forward, whose values no score has met, in LDS.
template <typename T> constexpr uint32_t kExponents = std::is_same_v<T, Bf16> ? 0x7f807f80u : 0x7c007c00u;
// bits 15 and 31: whether the numbers of a pair are not finite
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t pair) {
    return ((pair & kExponents<T>) + (std::is_same_v<T, Bf16> ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ bool any_not_finite(u32x4 x) {
    return (not_finite<T>(x[0]) | not_finite<T>(x[1]) | not_finite<T>(x[2]) | not_finite<T>(x[3])) != 0;
}
template <typename T>
__device__ __forceinline__ u32x4 only_finite(u32x4 x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] &= ~((not_finite<T>(x[i]) >> 15) * 0xffffu);
    return x;
}
// What is not finite of four numbers in LDS.  (Behind a wall, so that it takes few registers.)
template <typename T>
__device__ __forceinline__ f32x4 only_not_finite(const elem_t* from) {
    u32x2 x = *reinterpret_cast<const u32x2*>(from);
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] &= (not_finite<T>(x[i]) >> 15) * 0xffffu;
    asm volatile("" ::: "memory");
    return f32x4{T::to_float((elem_t)x[0]), T::to_float((elem_t)(x[0] >> 16)), T::to_float((elem_t)x[1]), T::to_float((elem_t)(x[1] >> 16))};
}

// A tile of 64 looped rows in LDS, and where this lane reads its operands (tile algebra: sjvp_ctx.hpp).  Rows are unpadded (D in 65 to 96 have rows
// of 128 columns) and the 16-byte pieces of a row are permuted by it, for both kinds of reads.  LDS serves 256 bytes a cycle: 16 lanes of a
// row-major read, so 16 neighbouring rows have to be in different places; and 32 lanes of a transposing read, which are four neighbouring rows of 64 bytes,
// so these four have to be too.  (The permutation of sjvp_device.hpp has the four rows in one or two places, for which the
// counters show six cycles lost to each transposing read of eight, half of the time that LDS was busy.)
//
// The places of a tile are LDS addresses in registers, which move to the tile's next place; what else differs from read to read is constant
// and stands in the instruction.
template <int HD>
struct SeqTile {
    static constexpr int kLd = HD == 96 ? 128 : HD, kElems = kCtxTile * kLd, kBytes = 2 * kElems, PP = kLd / 8;
    uint32_t row[HD / 16], lo[HD / 32], hi[HD / 32];

    static __device__ __forceinline__ int swz(int row) {
        if constexpr (kLd == 128) return (row & 3) << 2 | (row >> 2 & 3);
        if constexpr (kLd == 64) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
        return row >> 2 & 3;
    }
    __device__ __forceinline__ SeqTile(const elem_t* tile, int lane) {
        const uint32_t base = lds_addr(tile);
        const int y = lane & 31, h = lane >> 5, i16 = lane & 15;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) row[c] = base + 2 * (y * kLd + 8 * ((2 * c + h) ^ swz(y)));
        // within 16 lanes of a transposing read lane 4j + i supplies row j, columns 4i .. 4i+3, and lane n receives column n
        const int r = 4 * h + (i16 >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
#pragma unroll
        for (int z = 0; z < HD / 32; ++z) {
            lo[z] = base + 2 * (r * kLd + 8 * ((chunk + 4 * z) ^ swz(r)) + 4 * (i16 & 1));
            hi[z] = base + 2 * ((r + 8) * kLd + 8 * ((chunk + 4 * z) ^ swz(r + 8)) + 4 * (i16 & 1));
        }
    }
    __device__ __forceinline__ void move(int bytes) {
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) row[c] += bytes;
#pragma unroll
        for (int z = 0; z < HD / 32; ++z) lo[z] += bytes, hi[z] += bytes;
    }
    template <typename V>
    static __device__ __forceinline__ V __attribute__((address_space(3)))* at(uint32_t address) {
        return (V __attribute__((address_space(3)))*)address;
    }
    // A operand: 32 rows, chunk c of 16 columns.  from: bytes from the place to the first of the rows (whole multiples of 16 of them)
    __device__ __forceinline__ u32x4 rows(int from, int c) const { return *at<const u32x4>(row[c] + from); }
    // A operand of an output contraction: columns 32 dt .. 32 dt + 31 over 16 rows
    __device__ __forceinline__ u32x4 columns(int from, int dt) const {
        const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at<s16x4>(lo[dt] + from)));
        const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at<s16x4>(hi[dt] + from)));
        return u32x4{a[0], a[1], b[0], b[1]};
    }
    // scores of 32 rows and this lane's own row
    template <typename T>
    __device__ __forceinline__ f32x16 scores(int from, const u32x4* own, f32x16 s = {}) const {
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) s = Mma32<T>::run(rows(from, c), own[c], s);
        return s;
    }
    // OUT^T += A^T B for a score tile of 32 rows
    template <typename T>
    __device__ __forceinline__ void add_columns(f32x16* acc, int from, const f32x16& s) const {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const u32x4 b = pack_scores<T>(s, m);
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt) acc[dt] = Mma32<T>::run(columns(from + m * 16 * kLd * 2, dt), b, acc[dt]);
        }
    }
};

// A tile of 64 rows of a tensor on its way to LDS by NT threads: by LDS-DMA where rows start on 16-byte boundaries, through registers at any
// alignment otherwise.
template <int HD, bool DMA, int NT = kCtxThreads>
struct RowFeed {
    using At = SeqTile<HD>;
    static constexpr int PP = At::PP, N = kCtxTile * PP / NT;
    static_assert(kCtxTile * PP % NT == 0, "every thread copies whole pieces");
    u32x4 r[DMA ? 1 : N];
    uint32_t offset[N];

    __device__ __forceinline__ RowFeed(int64_t sl, int D, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = tid + NT * i, row = x / PP, c = x % PP;
            offset[i] = chunk_offset(row, 8 * (DMA ? c ^ At::swz(row) : c), sl, D);
        }
    }
    __device__ __forceinline__ void request(const elem_t* base, int64_t sl, int rows, int D, elem_t* place, int wave) {
        if constexpr (DMA) {
            const u32x4 from = rows_words(base, sl, rows, D);
            // (as TileFeed::request)
#pragma unroll
            for (int i = 0; i < N; ++i)
                asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                             :
                             : "v"(offset[i]), "s"(from), "s"(__builtin_amdgcn_readfirstlane(lds_addr(place) + 16 * (64 * wave + NT * i)))
                             : "memory");
        } else {
            const Rows from = make_rows(base, sl, rows, D);
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = read_chunk(from, offset[i]);
        }
    }
    __device__ __forceinline__ void deliver(elem_t* place, int D, int tid) {
        if constexpr (!DMA) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int x = tid + NT * i, row = x / PP, c = x % PP;
                if (D % 8) r[i] = chunk_shifted(r[i], 8 * c, D);
                *reinterpret_cast<u32x4*>(place + row * At::kLd + 8 * (c ^ At::swz(row))) = r[i];
            }
        }
    }
    static __device__ __forceinline__ void arrived() {
        if constexpr (DMA) __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    }
};

// Tiles of 64 keys and values on their way to LDS by four waves.  look() is called a tile ahead of request(), request() ahead of use,
// deliver() where the places are read next, behind it arrived() and a barrier.
// From a contiguous tensor (rows of a segment):
template <int HD, bool DMA>
struct SeqFeed {
    static constexpr bool kDma = DMA;
    RowFeed<HD, DMA> kf, vf;
    const elem_t *k, *v;
    __device__ __forceinline__ SeqFeed(const SeqParams& p, const SeqBlock& b, int hk, int tid)
        : kf(p.k.sl, p.D, tid), vf(p.v.sl, p.D, tid), k(p.k.head(0, hk) + b.token * p.k.sl), v(p.v.head(0, hk) + b.token * p.v.sl) {}
    __device__ __forceinline__ void look(const SeqParams&, int, int) {}
    __device__ __forceinline__ void request(const SeqParams& p, int t, int keys, elem_t* kp, elem_t* vp, int wave) {
        kf.request(k + (int64_t)t * kCtxTile * p.k.sl, p.k.sl, keys - t * kCtxTile, p.D, kp, wave);
        vf.request(v + (int64_t)t * kCtxTile * p.v.sl, p.v.sl, keys - t * kCtxTile, p.D, vp, wave);
    }
    __device__ __forceinline__ void deliver(const SeqParams& p, elem_t* kp, elem_t* vp, int tid) {
        kf.deliver(kp, p.D, tid), vf.deliver(vp, p.D, tid);
    }
    __device__ __forceinline__ void request_k(const SeqParams& p, int t, int keys, elem_t* kp, int wave) {
        kf.request(k + (int64_t)t * kCtxTile * p.k.sl, p.k.sl, keys - t * kCtxTile, p.D, kp, wave);
    }
    __device__ __forceinline__ void request_v(const SeqParams& p, int t, int keys, elem_t* vp, int wave) {
        vf.request(v + (int64_t)t * kCtxTile * p.v.sl, p.v.sl, keys - t * kCtxTile, p.D, vp, wave);
    }
    __device__ __forceinline__ void arrived() { kf.arrived(); }
};

// From the pages of a cache, 16-bit numbers (D is a multiple of 8 and rows are aligned): every lane of an LDS-DMA copy has an address of its
// own, so a tile may lie in any number of pages.
template <int HD>
struct PageFeed {
    using At = SeqTile<HD>;
    static constexpr bool kDma = true;
    static constexpr int CH = At::PP, N = kCtxTile * CH / kCtxThreads;
    int page[N], row[N];
    const int* table;
    int64_t head;
    int x;
    __device__ __forceinline__ PageFeed(const SeqParams& p, const SeqBlock& b, int hk, int tid)
        : table(p.pages.table + (b.segment - 1) * p.pages.table_stride), head(hk * p.pages.sh), x(tid) {}
    __device__ __forceinline__ void look(const SeqParams& p, int t, int keys) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int key = t * kCtxTile + (x + kCtxThreads * i) / CH, at = p.pages.page_of(key);
            page[i] = key < keys ? table[at] : -1;
            row[i] = key - at * p.pages.size;
        }
    }
    __device__ __forceinline__ void request(const SeqParams& p, int, int, elem_t* kp, elem_t* vp, int wave) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (x + kCtxThreads * i) / CH, c = (x + kCtxThreads * i) % CH ^ At::swz(r);
            const bool ok = (uint32_t)page[i] < (uint32_t)p.pages.pages && 8 * c < p.D;
            const int64_t at = p.pages.at(page[i], row[i]) + head + 16 * c;
            const void* none = &kZeroPiece;
            const void *from_k = ok ? p.pages.k + at : none, *from_v = ok ? p.pages.v + at : none;
            dma16(from_k, lds_addr(kp) + 16 * (64 * wave + kCtxThreads * i));
            dma16(from_v, lds_addr(vp) + 16 * (64 * wave + kCtxThreads * i));
        }
    }
    __device__ __forceinline__ void deliver(const SeqParams&, elem_t*, elem_t*, int) {}
    __device__ __forceinline__ void arrived() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)
};

// From pages of 8-bit numbers (D is a multiple of 16), which become 16-bit ones on their way, once for the four waves.
template <typename T, int HD>
struct PageFeed8 {
    using At = SeqTile<HD>;
    static constexpr bool kDma = false;
    static constexpr int PC = HD / 16, N = (kCtxTile * PC + kCtxThreads - 1) / kCtxThreads;
    u32x4 kr[N], vr[N];
    uint32_t ks[N], vs[N];
    int page[N], row[N];
    const int* table;
    int64_t head, scale_head;
    int x;
    __device__ __forceinline__ PageFeed8(const SeqParams& p, const SeqBlock& b, int hk, int tid)
        : table(p.pages.table + (b.segment - 1) * p.pages.table_stride), head(hk * p.pages.sh), scale_head(hk * p.pages.scale_sh), x(tid) {}
    __device__ __forceinline__ void look(const SeqParams& p, int t, int keys) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (x + kCtxThreads * i) / PC, key = t * kCtxTile + r, at = p.pages.page_of(key);
            page[i] = r < kCtxTile && key < keys ? table[at] : -1;
            row[i] = key - at * p.pages.size;
        }
    }
    __device__ __forceinline__ void request(const SeqParams& p, int, int, elem_t*, elem_t*, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (x + kCtxThreads * i) % PC;
            const bool ok = (uint32_t)page[i] < (uint32_t)p.pages.pages && 16 * c < p.D;
            const int64_t at = p.pages.at(page[i], row[i]) + head + 16 * c;
            const int64_t sat = p.pages.scale_at(page[i], row[i]) + scale_head + c / 2;
            const void* none = &kZeroPiece;
            kr[i] = global<u32x4>(ok ? p.pages.k + at : none), vr[i] = global<u32x4>(ok ? p.pages.v + at : none);
            ks[i] = global<uint8_t>(ok ? p.pages.ks + sat : none), vs[i] = global<uint8_t>(ok ? p.pages.vs + sat : none);
        }
    }
    __device__ __forceinline__ void deliver(const SeqParams&, elem_t* kp, elem_t* vp, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int y = x + kCtxThreads * i, r = y / PC, c = y % PC;
            if (kCtxTile * PC % kCtxThreads && y >= kCtxTile * PC) break;
            const float a = scale_of(ks[i]), b = scale_of(vs[i]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int at = r * At::kLd + 8 * ((2 * c + j) ^ At::swz(r));
                *reinterpret_cast<u32x4*>(kp + at) = from_e4m3_8<T>(kr[i][2 * j], kr[i][2 * j + 1], a);
                *reinterpret_cast<u32x4*>(vp + at) = from_e4m3_8<T>(vr[i][2 * j], vr[i][2 * j + 1], b);
            }
        }
    }
    __device__ __forceinline__ void arrived() {}
};

// Running maximum and sum of a row, as in the attention on keys of another length: raised only past 2^8.
template <int HD>
struct SeqSums {
    f32x16 acc[HD / 32];
    float m, ref, l;  // maximum (-inf: no key yet), what is subtracted (finite), sum of this lane's half

    __device__ __forceinline__ SeqSums() : acc{}, m(-INFINITY), ref(0.0f), l(0.0f) {}

    // The rows' maxima with the scores of 32 N keys; keys from `left` on are not seen (masked).
    template <bool MASKED, int N>
    __device__ __forceinline__ void raise(f32x16 (&s)[N], float c, int left, int h) {
        if constexpr (MASKED) {
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
        top *= c;
        if (__builtin_amdgcn_ballot_w64(top > m + 8.0f)) {
            const float grown = fmaxf(m, halves_max(top));
            const float now = grown == -INFINITY ? 0.0f : grown;
            const float f = m == -INFINITY ? 1.0f : fast_exp2(ref - now);  // (no sums yet but infinities, of the careful tiles)
            m = grown, ref = now;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt) acc[dt] *= f;
        }
    }
    template <int N>
    __device__ __forceinline__ void exponentials(f32x16 (&s)[N], float c) {
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = fast_exp2(__builtin_fmaf(s[u][r], c, -ref));
                sum += s[u][r];
            }
        l += sum;
    }
    template <bool MASKED, int N>
    __device__ __forceinline__ void take(f32x16 (&s)[N], float c, int left, int h) {
        raise<MASKED>(s, c, left, h);
        exponentials(s, c);
    }
};

// Of a tile of 64 rows: out += factor times what is not finite of the rows [first, end); the finite numbers alone.
template <typename T, int HD>
__device__ __forceinline__ void add_not_finite(f32x16* out, const elem_t* tile, int first, int end, float factor, int h) {
    for (int j = first; j < end; ++j) {
        const elem_t* from = tile + j * SeqTile<HD>::kLd + 4 * h;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
            const f32x4 more = only_not_finite<T>(from + 8 * (c ^ SeqTile<HD>::swz(j)));
#pragma unroll
            for (int i = 0; i < 4; ++i) out[c / 4][4 * (c % 4) + i] = __builtin_fmaf(factor, more[i], out[c / 4][4 * (c % 4) + i]);
        }
    }
}
template <typename T, int HD, int NT>
__device__ __forceinline__ void keep_finite(elem_t* tile, int tid) {
    for (int x = tid; x < SeqTile<HD>::kElems / 8; x += NT) {
        u32x4* piece = reinterpret_cast<u32x4*>(tile) + x;
        *piece = only_finite<T>(*piece);
    }
}

// Sums of a wave's own 32 rows, OUT^T, as rows in memory whose places `at` gives, through the wave's own LDS region of [32][HD + 8].
template <typename T, int HD, typename F>
__device__ __forceinline__ void store_rows_at(const f32x16* acc, float factor, int rows, elem_t* region, int lane, int D, F&& at) {
    elem_t* mine = region + (lane & 31) * (HD + 8) + 4 * (lane >> 5);
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = factor == 0.0f ? 0.0f : acc[dt][4 * i + j] * factor;  // (sums of rows without a result may be NaN)
            *reinterpret_cast<u32x2*>(mine + 32 * dt + 8 * i) = u32x2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
        }
    wave_exchange();
    constexpr int CH = HD / 8;
#pragma unroll
    for (int x0 = 0; x0 < 32 * CH; x0 += 64) {
        const int x = x0 + lane, row = x / CH, c8 = 8 * (x % CH);
        if (row < rows) store_chunk(at(row), *reinterpret_cast<const u32x4*>(region + row * (HD + 8) + c8), c8, D);
    }
    wave_exchange();
}

}  // namespace sjvp
