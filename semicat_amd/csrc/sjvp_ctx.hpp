// Attention of queries on keys of another length, and with a learned relative position bias: parameters and device
// building blocks (kernels: sjvp_ctx_fwd.hpp, sjvp_ctx_bwd.hpp).
//
//   s[i][j] = scale q_i.k_j + table[bucket(j - (start + i))][head]     for j < key length (and j <= start + i if causal)
//   lse_i = log sum_j exp s[i][j],  p = exp(s - lse),  o_i = sum_j p[i][j] v_j
//
// A query head reads key head  head / (Hq / Hkv).  A row that sees no key has o = 0 and no gradient.
//
// Tile algebra (v_mfma_f32_32x32x16_{bf16,f16}): C[y][x] += sum_k A[y][k] B[k][x] with
//     A: lane l holds row y = l % 32, k = 8*(l/32) + i (i < 8);   B: column x = l % 32, same k;
//     C: lane l holds column x = l % 32 and, in register r < 16, row y = 8*(r/4) + 4*(l/32) + r%4.
// A wave owns 32 positions as columns, one to a lane pair (l, l + 32), so that the softmax statistics of a row are one
// register each and a reduction over the looped axis is register arithmetic and one exchange of the halves.  Its
// operands (B) stay in registers, the looped side is A from LDS.  Registers 8m .. 8m+7 of a score tile, rounded to 16
// bits, are the B operand of the next contraction under the numbering  k = 8h + i  <->  y = 16m + 8*(i/4) + 4h + i%4  (h = l/32);
// A in that numbering is what two transposing LDS reads of four rows deliver.
#pragma once
#include <type_traits>

#include "sjvp_device.hpp"
#include "../../include/sjvp.h"

namespace sjvp {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kCtxWaves = 4;
constexpr int kCtxThreads = 64 * kCtxWaves;
constexpr int kCtxOwned = 32 * kCtxWaves;  // owned positions of a workgroup whose waves share their tiles
constexpr int kCtxTile = 64;               // looped positions per tile
constexpr int kCtxPad = 64;                // entries of the bias row beyond the last single distance, on each side
constexpr int kCtxStats = 2 * 3 * kCtxTile; // floats of LDS for what the column-owned launches keep of two tiles' rows
constexpr int kCtxBuckets = SJVP_CTX_MAX_BUCKETS;
constexpr int kCtxMost = 1 << 29;          // positions and lengths: sums of three stay within 32 bits

template <typename T> struct Mma32;
template <> struct Mma32<Bf16> {
    static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma32<Fp16> {
    static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

struct CtxView {
    elem_t* ptr;
    int64_t sb, sh, sl;
    __device__ __forceinline__ elem_t* head(int b, int h) const { return ptr + b * sb + h * sh; }
};

struct CtxParams {
    CtxView q, k, v, o, rest, g, dq, dk, dv;  // rest: what the rounding of o left (or null); g: the cotangent of o
    float *lse, *folded;                     // [B,Hq,Lq][2]: (m, l) of each row; [3][B,Hq,Lq]: row_stat_folded, -delta
    float *part, *stat;                      // sums of split work: rows of HD floats; their (maximum, sum) pairs
    float* tpart;                            // bucket sums of each workgroup
    void* dtable;
    const void* table;
    const int *klen, *qlen, *start;          // per batch entry, or null
    int64_t tsb, tsh, dtsb, dtsh;            // strides of table and dtable (bucket, head)
    int start0, table_type;
    int B, Hq, Hkv, G, Lq, Lk, D;
    float scale, c;                          // c = scale * log2(e)
    int buckets, both, causal, far;          // buckets of a direction; far: the first distance of the last one
    int splits, blocks;                      // splits of the looped axis; workgroups of a split over the owned axis
    int packed;                              // ctx_fwd_few: heads to a block of rows; ctx_bwd_one: sets of dS tiles
    int cols;                                // ctx_sum: dK and dV, not dQ
    alignas(4) uint16_t first[kCtxBuckets];  // first distance of each bucket
};

// max / sum over the two lanes of a column
__device__ __forceinline__ float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// the values of other lanes, by a DPP pattern
template <int PATTERN>
__device__ __forceinline__ float lanes_turned(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), PATTERN, 0xf, 0xf, false));
}
// sum over 16 neighbouring lanes, in all of them
__device__ __forceinline__ float sum16(float x) {
    x += lanes_turned<0x128>(x);  // turned by 8 of 16
    x += lanes_turned<0x124>(x);
    x += lanes_turned<0x122>(x);
    return x + lanes_turned<0x121>(x);
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Rows start on element boundaries; 16-byte accesses need no more.  Where a row ends inside a chunk of eight columns (D is not a
// multiple of 8), the chunk is taken from the row's last eight elements and moved down: no access leaves the row.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
__device__ __forceinline__ int chunk_column(int c8, int D) { return min(c8, D - 8); }
__device__ __forceinline__ u32x4 chunk_shifted(u32x4 x, int c8, int D) {
    const int over = c8 + 8 - D;  // elements of the chunk beyond the row
    if (over <= 0) return x;
    return __builtin_bit_cast(u32x4, __builtin_bit_cast(unsigned __int128, x) >> (16 * min(over, 7)));
}
// Eight elements of a row from column c8 on, zeros beyond D.
__device__ __forceinline__ u32x4 load_chunk(const elem_t* p, int c8, int D) {
    if (c8 >= D) return u32x4{0u, 0u, 0u, 0u};
    const u32x4 x = *reinterpret_cast<const u32x4_any*>(p + chunk_column(c8, D));
    return D % 8 ? chunk_shifted(x, c8, D) : x;
}
__device__ __forceinline__ void store_chunk(elem_t* p, u32x4 x, int c8, int D) {
    if (c8 + 8 <= D) {
        *reinterpret_cast<u32x4_any*>(p + c8) = x;
    } else if (c8 < D) {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (c8 + i < D) p[c8 + i] = (elem_t)(x[i / 2] >> (16 * (i % 2)));
    }
}

// Four elements of a row from column c4 on.
typedef u32x2 __attribute__((aligned(2))) u32x2_any;
__device__ __forceinline__ void store_quad(elem_t* p, u32x2 x, int c4, int D) {
    if (c4 + 4 <= D) {
        *reinterpret_cast<u32x2_any*>(p + c4) = x;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (c4 + i < D) p[c4 + i] = (elem_t)(x[i / 2] >> (16 * (i % 2)));
    }
}

// B operands of this lane's own row (all chunks of 16 of the head dimension), from memory.
template <int HD>
__device__ __forceinline__ void own_operands(u32x4* out, const elem_t* row, bool ok, int h, int D) {
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) out[c] = ok ? load_chunk(row, 16 * c + 8 * h, D) : u32x4{0u, 0u, 0u, 0u};
}

// A tile of looped rows in LDS, and where this lane reads its operands.  Tiles that come through registers are [64][HD + 8]: the 16
// bytes between rows spread both the row-major 16-byte reads of 16 rows and the transposing reads of 4 rows over all banks.
// LDS-DMA copies leave no gaps: there the 16-byte pieces of a row are permuted instead (swz).
template <int HD, bool DMA>
struct Tile {
    static constexpr int kLd = DMA ? HD : HD + 8, kElems = kCtxTile * kLd;
    int row[HD / 16], col[HD == 32 ? 2 : HD / 32];

    __device__ __forceinline__ explicit Tile(int lane) {
        const int y = lane & 31, h = lane >> 5, i16 = lane & 15;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) row[c] = DMA ? y * HD + 8 * ((2 * c + h) ^ swz<HD>(y)) : y * kLd + 16 * c + 8 * h;
        // within 16 lanes of a transposing read lane 4j + i supplies row j, columns 4i .. 4i+3, and lane n receives column n
        const int r = 4 * h + (i16 >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
#pragma unroll
        for (int z = 0; z < (HD == 32 ? 2 : HD / 32); ++z)
            col[z] = DMA ? r * HD + 8 * (chunk ^ swz<HD>(r) ^ (HD == 32 ? 2 * z : 4 * z)) + 4 * (i16 & 1) : r * kLd + 8 * chunk + 4 * (i16 & 1);
    }
    // A operand: rows row0 .. row0 + 31 (row0 a multiple of 32), chunk c of 16 columns
    __device__ __forceinline__ u32x4 rows(const elem_t* tile, int row0, int c) const {
        return *reinterpret_cast<const u32x4*>(tile + row0 * kLd + row[c]);
    }
    // A operand of an output contraction: columns 32 dt .. 32 dt + 31 (as rows of A) over the 16 rows from row0 on (a multiple of
    // 16), in the numbering at the top
    __device__ __forceinline__ u32x4 columns(const elem_t* tile, int row0, int dt) const {
        // the permutation of rows 8 further differs in one bit, and so does the place of the next 32 columns
        const elem_t *p = tile + row0 * kLd, *lo, *hi;
        if constexpr (DMA) {
            lo = p + col[HD == 32 ? 0 : dt];
            hi = p + 8 * kLd + col[HD == 32 ? 1 : HD == 64 ? dt ^ 1 : dt ^ 2];
        } else {
            lo = p + col[0] + 32 * dt;
            hi = lo + 8 * kLd;
        }
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lo)));
        const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(hi)));
        return u32x4{a[0], a[1], b[0], b[1]};
    }
};

// Registers 8m .. 8m+7 of a score tile as a B operand.
template <typename T>
__device__ __forceinline__ u32x4 pack_scores(const f32x16& s, int m) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = T::pack2(s[8 * m + 2 * i], s[8 * m + 2 * i + 1]);
    return r;
}

// Rows of a tensor from a given one on, as a buffer: reads behind the last row that exists return zeros (whatever memory holds there),
// with no branch.  Offsets are 32 bits within a tile, so the host keeps row strides below 2^24 elements.
constexpr uint32_t kNoChunk = 0x80000000u;  // an offset behind every buffer
__device__ __forceinline__ int rows_bytes(int64_t sl, int rows, int D) {
    return rows > 0 ? 2 * ((min(rows, kCtxTile) - 1) * (int)sl + D) : 0;
}
typedef __amdgpu_buffer_rsrc_t Rows;
constexpr int kRowsFlags = 0x00020000;
__device__ __forceinline__ Rows make_rows(const elem_t* base, int64_t sl, int rows, int D) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<elem_t*>(base), 0, rows_bytes(sl, rows, D), kRowsFlags);
}
// the four words of that descriptor
__device__ __forceinline__ u32x4 rows_words(const elem_t* base, int64_t sl, int rows, int D) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    return u32x4{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, (uint32_t)rows_bytes(sl, rows, D), (uint32_t)kRowsFlags};
}
__device__ __forceinline__ uint32_t chunk_offset(int row, int c8, int64_t sl, int D) {
    return c8 < D ? 2u * (uint32_t)(row * (int)sl + chunk_column(c8, D)) : kNoChunk;
}
__device__ __forceinline__ u32x4 read_chunk(Rows rows, uint32_t offset) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0));
}

// A tile of 64 rows on its way from memory to LDS by NT threads: straight into LDS where rows start on 16-byte boundaries (DMA), through
// registers at any alignment otherwise.  request() is called ahead, deliver() where the place is read next, behind it arrived()
// and a barrier.
template <int HD, bool DMA, int NT = kCtxThreads>
struct TileFeed {
    static constexpr int CH = HD / 8;
    static constexpr int N = kCtxTile * CH / NT;
    static_assert(kCtxTile * CH % NT == 0, "every thread copies whole chunks");
    u32x4 r[DMA ? 1 : N];
    uint32_t offset[N];

    __device__ __forceinline__ TileFeed(int64_t sl, int D, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = tid + NT * i, row = x / CH, c = x % CH;
            offset[i] = chunk_offset(row, 8 * (DMA ? c ^ swz<HD>(row) : c), sl, D);
        }
    }
    __device__ __forceinline__ void request(const elem_t* base, int64_t sl, int rows, int D, elem_t* place, int wave) {
        if constexpr (DMA) {
            const u32x4 from = rows_words(base, sl, rows, D);
            // M0 carries the LDS address; nothing else here uses it.  Counted by vmcnt, unknown to the compiler: its own waits for loads
            // are stricter for it, never laxer, since loads return in order.
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
                const int x = tid + NT * i;
                if (D % 8) r[i] = chunk_shifted(r[i], 8 * (x % CH), D);
                *reinterpret_cast<u32x4*>(place + (x / CH) * Tile<HD, DMA>::kLd + 8 * (x % CH)) = r[i];
            }
        }
    }
    static __device__ __forceinline__ void arrived() {
        if constexpr (DMA) __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    }
};

// The bucket of a position difference (key minus query): the last bucket whose first distance is not beyond the distance;
// differences above zero have distances and buckets of their own (`both`) or distance 0.  The first distances are the same for all
// lanes and come as scalars, so counting them is quicker than a search, whose every step would wait for memory.
__device__ __forceinline__ int ctx_bucket(const CtxParams& p, int rel) {
    const int d = p.both ? abs(rel) : max(-rel, 0);
    int bucket = -1;
    for (int i = 0; i < p.buckets; i += 2) {
        const uint32_t two = reinterpret_cast<const uint32_t*>(p.first)[i / 2];
        bucket += (d >= (int)(two & 0xffffu)) + (i + 1 < p.buckets && d >= (int)(two >> 16));
    }
    return bucket + (p.both && rel > 0 ? p.buckets : 0);
}

__device__ __forceinline__ float ctx_table(const CtxParams& p, int bucket, int head) {
    const int64_t at = bucket * p.tsb + head * p.tsh;
    if (p.table_type == SJVP_FP32) return reinterpret_cast<const float*>(p.table)[at];
    const elem_t x = reinterpret_cast<const elem_t*>(p.table)[at];
    return p.table_type == SJVP_BF16 ? Bf16::to_float(x) : Fp16::to_float(x);
}

__device__ __forceinline__ int ctx_all_buckets(const CtxParams& p) { return p.both ? 2 * p.buckets : p.buckets; }
__device__ __forceinline__ int ctx_row_entries(const CtxParams& p) { return 2 * (p.far + kCtxPad) + 1; }

// The bias of a head (of `heads` from it on, one row after another) by position difference, entry far + pad for difference 0, in units
// of log2; -inf for keys behind a causal query, so that the kernels need no other mask for these.  A table entry near the lowest
// float32 would leave the range with the factor log2(e); it is raised to -2.3e38, still below any score.  NaN stays.
// (An entry's bucket serves all heads: filled head by head, eight heads of B=4 Lq=2 Lk=4096 D=64 took 16.9 us in place of 12.1.)
__device__ __forceinline__ void fill_bias_row(const CtxParams& p, float* row, int head, int tid, int threads, int heads = 1) {
    const int entries = ctx_row_entries(p);
    for (int x = tid; x < entries; x += threads) {
        const int rel = x - p.far - kCtxPad, bucket = ctx_bucket(p, rel);
        for (int i = 0; i < heads; ++i) {
            const float t = ctx_table(p, bucket, head + i);
            row[i * entries + x] = t == -INFINITY || (p.causal && rel > 0) ? -INFINITY : (t < -2.3e38f ? -2.3e38f : t) * kLog2e;
        }
    }
}

struct CtxBatch {
    int keys, rows, start;  // key length, query length, position of query 0
    __device__ __forceinline__ CtxBatch(const CtxParams& p, int b)
        : keys(p.klen ? min(max(p.klen[b], 0), p.Lk) : p.Lk),
          rows(p.qlen ? min(max(p.qlen[b], 0), p.Lq) : p.Lq),
          start(min(max(p.start ? p.start[b] : 0, -kCtxMost), kCtxMost) + p.start0) {}
    // whether some row sees more than one key: otherwise the scores have no gradient at all
    __device__ __forceinline__ bool any_scored(const CtxParams& p) const { return keys != 1 && !(p.causal && start + rows <= 1); }
    // keys that the row sees
    __device__ __forceinline__ int seen(const CtxParams& p, int row) const {
        return p.causal ? max(0, min(keys, start + row + 1)) : keys;
    }
};

// The statistics of a row: m, which its scores (in units of log2) have subtracted, and l, the sum of their exponentials then.  Two numbers, since
// m + log2 l in one would lose l beside a large m (1e8: P would be 1 for every key in place of 1/n).  No key: both are zero.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef f32x2 __attribute__((aligned(4))) f32x2_any;
__device__ __forceinline__ void store_stat(const CtxParams& p, int64_t place, float m, float l) {
    if (p.lse) *reinterpret_cast<f32x2_any*>(p.lse + 2 * place) = f32x2{l == 0.0f ? 0.0f : m, l};
}
__device__ __forceinline__ f32x2 load_stat(const CtxParams& p, int64_t place) { return *reinterpret_cast<const f32x2_any*>(p.lse + 2 * place); }
// What a backward subtracts from the row's scores, and what it multiplies the exponentials with; none of them is left in a row without keys.
__device__ __forceinline__ f32x2 row_stat(f32x2 stat) {
    return stat[1] == 0.0f ? f32x2{INFINITY, 0.0f} : f32x2{stat[0], 1.0f / stat[1]};
}
// The same for launches that walk the rows, where a factor takes reads and registers (in the single backward launch, B=64 H=12 Lq=128 Lk=256
// forward and backward, 87 us in place of 72): it is 1 where m + log2 l is below 64, and its rounding below 1.4e-6 of P.
__device__ __forceinline__ f32x2 row_stat_folded(f32x2 stat) {
    if (stat[1] == 0.0f) return f32x2{INFINITY, 1.0f};
    const float both = stat[0] + fast_log2(stat[1]);
    return fabsf(both) < 64.0f ? f32x2{both, 1.0f} : row_stat(stat);
}

// Workgroups run on XCD blockIdx % 8.  The workgroups of one (batch, key head) unit read the same rows: each XCD takes every
// eighth unit as a whole and finds them in its L2, and batch entries of different lengths spread over all XCDs.  With few units
// that do not divide by eight the XCDs would differ in load, and the plain order stays.
struct CtxWork {
    int unit, inner;
    bool some;
};
inline __host__ __device__ bool ctx_by_xcd(int64_t units) { return units % 8 == 0 || units >= 64; }
inline __host__ __device__ int64_t ctx_grid(int64_t units, int64_t inner) {
    return (ctx_by_xcd(units) ? (units + 7) / 8 * 8 : units) * inner;
}
__device__ __forceinline__ CtxWork ctx_work(int units, int inner) {
    const int x = blockIdx.x;
    if (!ctx_by_xcd(units)) return {x / inner, x % inner, true};
    const int slot = x >> 3, unit = (x & 7) + 8 * (slot / inner);
    return {unit, slot % inner, unit < units};
}

// What the rounding of two numbers to w left of them, as it stands in memory beside o.  fp16: the difference, 2^11 times as large (at most as
// large as the number then), which makes 22 bits in all and, for small numbers, steps of 2^-35; bf16, where the difference would make 17: the
// difference of the bits as a signed number, which makes all 24.
constexpr float kRestScale = 2048.0f;
template <typename T>
__device__ __forceinline__ uint32_t rest_of(uint32_t w, float lo, float hi) {
    if constexpr (!std::is_same_v<T, Bf16>) return T::pack2((lo - T::to_float((elem_t)w)) * kRestScale, (hi - T::to_float((elem_t)(w >> 16))) * kRestScale);
    const auto bits = [](float x, uint32_t top) {
        return (uint32_t)min(max((int)(__float_as_uint(x) - top), -32768), 32767);
    };
    return (bits(lo, w << 16) & 0xffffu) | bits(hi, w & 0xffff0000u) << 16;
}
template <typename T>
__device__ __forceinline__ float with_rest(elem_t o, elem_t rest) {
    if constexpr (!std::is_same_v<T, Bf16>) return __builtin_fmaf(T::to_float(rest), 1.0f / kRestScale, T::to_float(o));
    return __uint_as_float(((uint32_t)o << 16) + (uint32_t)(int)(int16_t)rest);
}

// Sums of a wave's own 32 rows, OUT^T (row of C: column of the result), as rows in memory: through the wave's own LDS region of
// [32][HD + 8], so that rows go out in pieces of 16 bytes.  `rest`: what the rounding leaves of them.
template <typename T, int HD>
__device__ __forceinline__ void store_rows(const f32x16* acc, float factor, elem_t* out, int64_t sl, int rows, elem_t* region,
                                           int lane, int D, bool rest = false) {
    const int h = lane >> 5;
    elem_t* mine = region + (lane & 31) * (HD + 8) + 4 * h;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[4];
            uint32_t w[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = factor == 0.0f ? 0.0f : acc[dt][4 * i + j] * factor;  // (sums of rows without a result may be NaN)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                w[j] = T::pack2(x[2 * j], x[2 * j + 1]);
                if (rest) w[j] = rest_of<T>(w[j], x[2 * j], x[2 * j + 1]);
            }
            *reinterpret_cast<u32x2*>(mine + 32 * dt + 8 * i) = u32x2{w[0], w[1]};
        }
    wave_exchange();
    constexpr int CH = HD / 8;
#pragma unroll
    for (int x0 = 0; x0 < 32 * CH; x0 += 64) {
        const int x = x0 + lane, row = x / CH, c8 = 8 * (x % CH);
        if (row < rows) store_chunk(out + row * sl, *reinterpret_cast<const u32x4*>(region + row * (HD + 8) + c8), c8, D);
    }
    wave_exchange();
}

// The same sums as fp32 rows of HD, for a later launch to add up; zeros for a lane that has no result.
template <int HD>
__device__ __forceinline__ void store_part(const f32x16* acc, bool some, float* out, int rows, int lane) {
    if ((lane & 31) >= rows) return;
    float* mine = out + (int64_t)(lane & 31) * HD + 4 * (lane >> 5);
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(mine + 32 * dt + 8 * i) =
                some ? f32x4{acc[dt][4 * i], acc[dt][4 * i + 1], acc[dt][4 * i + 2], acc[dt][4 * i + 3]} : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// Where the position differences of a tile lie: all beyond `far` on one side, which has one bias, or not.  Looped positions are walked in
// order, so that the tiles of each kind follow each other and each kind has a loop of its own, without a branch in its body.
enum CtxBand { kBelow, kNear, kAbove };
template <CtxBand B> using InBand = std::integral_constant<CtxBand, B>;
// whole tiles in front of a position, of `tiles`
__device__ __forceinline__ int tiles_before(int position, int tiles) { return min(max(position, 0) / kCtxTile, tiles); }

// First entry of a bias row (or of sums by difference) for a lane or a wave that uses `count` from it on: differences wholly beyond `far`
// have the same bias, so that their entries may be taken from the row's ends.
__device__ __forceinline__ int row_entry(const CtxParams& p, int rel, int count) {
    return min(max(rel + p.far + kCtxPad, 0), ctx_row_entries(p) - count);
}

// Whether a bias (in units of log2) is such that rounding score plus bias shows in the probabilities: 2^-14 from 2^10 on, and nothing is left of
// the scores in the end (lowest numbers as masks).  Tiles of one bias subtract the maximum from the bias and round only then, so those with
// such a bias go through the loop near the diagonal, which reads the ends of the bias row: every launch forms the same scores.
__device__ __forceinline__ bool ctx_rounds(float bias) {
    const float x = fabsf(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(bias))));
    return x >= 1024.0f && x < INFINITY;
}

// OUT^T += A^T B for the two halves of a packed score tile whose looped rows start at row0 of the tile.
template <typename T, int HD, bool DMA>
__device__ __forceinline__ void add_columns(f32x16* acc, const Tile<HD, DMA>& at, const elem_t* tile, int row0, const f32x16& s) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const u32x4 b = pack_scores<T>(s, m);
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
            acc[dt] = Mma32<T>::run(at.columns(tile, row0 + 16 * m, dt), b, acc[dt]);
    }
}

// The same with what the rounding of the scores leaves: TERMS roundings of 8 (bf16) or 11 bits each.
template <typename T, int TERMS, int HD, bool DMA>
__device__ __forceinline__ void add_columns_exact(f32x16* acc, const Tile<HD, DMA>& at, const elem_t* tile, int row0, const f32x16& s) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        u32x4 b[TERMS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo = s[8 * m + 2 * i], hi = s[8 * m + 2 * i + 1];
#pragma unroll
            for (int x = 0; x < TERMS; ++x) {
                b[x][i] = T::pack2(lo, hi);
                lo -= T::to_float((elem_t)b[x][i]), hi -= T::to_float((elem_t)(b[x][i] >> 16));
            }
        }
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) {
            const u32x4 a = at.columns(tile, row0 + 16 * m, dt);
#pragma unroll
            for (int x = 0; x < TERMS; ++x) acc[dt] = Mma32<T>::run(a, b[x], acc[dt]);
        }
    }
}

template <typename T, int HD, bool DMA>
__device__ __forceinline__ f32x16 scores(const Tile<HD, DMA>& at, const elem_t* tile, int row0, const u32x4* own, f32x16 s = {}) {
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) s = Mma32<T>::run(at.rows(tile, row0, c), own[c], s);
    return s;
}

// looped row of register r of a score tile
__device__ __forceinline__ int tile_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

}  // namespace sjvp
