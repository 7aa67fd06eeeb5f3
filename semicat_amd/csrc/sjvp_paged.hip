// Pages of a cache written and read back (sjvp_seq.hpp has their layout).
//
// Writing in 8 bits: 32 columns of a row share a power of two 2^e, the least one by which none of their finite numbers goes beyond 448, the
// largest e4m3 number, within the exponents for which every number that the 8 bits stand for is one of the cache's own type.  Scaling
// by a power of two is exact, so the only rounding is the one to e4m3 (to nearest even), and reading back rounds nothing.  What is not
// finite becomes NaN.  At the largest exponent numbers end at 240: the next one, 256, is none of the type's.
#include "sjvp_seq_launch.hpp"

namespace sjvp {

// The segment that holds a token: the last one that does not begin behind it.  (Of offsets that descend it may begin behind the token or end before it.)
__device__ __forceinline__ int seq_segment(const SeqParams& p, int token, int lane) {
    int lo = 0, hi = p.B + 2;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, x = lo + lane * step;
        const int n = __popcll(__builtin_amdgcn_ballot_w64(lane == 0 || (x < hi && seq_offset(p, x) <= token)));
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

template <typename T> constexpr int kScaleLow = std::is_same_v<T, Bf16> ? -117 : -15;
template <typename T> constexpr int kScaleHigh = std::is_same_v<T, Bf16> ? 120 : 8;

__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
    return bits < 0x7f800000u ? bits : 0u;
}

// 16 columns to 8 bits, by this lane and the neighbour that has the other 16 of a group; the group's exponent code.
template <typename T>
__device__ __forceinline__ uint32_t to_e4m3(u32x4 a, u32x4 b, u32x4& codes) {
    float x[16];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w = i < 4 ? a[i] : b[i - 4];
        x[2 * i] = T::to_float((elem_t)w), x[2 * i + 1] = T::to_float((elem_t)(w >> 16));
        most = max(most, max(finite_bits(x[2 * i]), finite_bits(x[2 * i + 1])));
    }
    most = max(most, __float_as_uint(lanes_turned<0xB1>(__uint_as_float(most))));  // lanes 1, 0, 3, 2 of four
    // most = 1.f 2^(E - 127) <= 448 2^e = 1.75 2^(8 + e)
    const int e = min(max((int)(most >> 23) - 135 + ((most & 0x7fffffu) > 0x600000u), kScaleLow<T>), kScaleHigh<T>);
    const float inverse = __uint_as_float((uint32_t)(127 - e) << 23), top = e == kScaleHigh<T> ? 240.0f : 448.0f;
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const bool finite = (__float_as_uint(x[i]) & 0x7f800000u) != 0x7f800000u;
        y[i] = finite ? fminf(fmaxf(x[i] * inverse, -top), top) : __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        codes[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false), true);
    return (uint32_t)(e + 127);
}

// A wave writes one token: its rows of K and V of all heads, 16 bytes of a page to a lane.  A lane quantises 16 columns, so that a group of 32 needs one
// exchange.  Eight prompts of 2048 to 4096 tokens, 8 heads of 128, e4m3: 28 us = 5.4 TB/s, the vector unit busy all the while; one token each
// of 64 sequences: 4.5 us, those of any launch.
template <typename T, bool E4M3>
__global__ __launch_bounds__(kCtxThreads) void paged_write(SeqParams p) {
    const int lane = threadIdx.x & 63, token = __builtin_amdgcn_readfirstlane(blockIdx.x * kCtxWaves + (threadIdx.x >> 6));
    if (token >= p.T) return;
    const int segment = seq_segment(p, token, lane);
    if (segment < 1 || segment > p.B) return;
    const int first = seq_offset(p, segment), end = seq_offset(p, segment + 1), length = max(p.lengths[segment - 1], 0);
    if (token < first || token >= end) return;  // (offsets that descend; a position would lie behind the length, and its page outside the table)
    const int position = length - (end - first) + token - first;
    if (position < 0 || position >= p.pages.capacity) return;
    const int at = p.pages.page_of(position), page = p.pages.table[(segment - 1) * p.pages.table_stride + at], row = position - at * p.pages.size;
    if ((uint32_t)page >= (uint32_t)p.pages.pages) return;
    constexpr int kColumns = E4M3 ? 16 : 8;
    const int per = E4M3 ? (p.D + 31) / 32 * 2 : p.D / 8;  // (E4M3: the lanes of a group stand side by side)
    const int64_t to = p.pages.at(page, row), scale_to = p.pages.scale_at(page, row);
    for (int x0 = 0; x0 < 2 * p.Hkv * per; x0 += 64) {
        const int x = x0 + lane, unit = x % per, hx = x / per, v = hx >= p.Hkv, head = v ? hx - p.Hkv : hx, c = kColumns * unit;
        const bool ok = hx < 2 * p.Hkv && c < p.D;
        const elem_t* from = (v ? p.v : p.k).head(0, head) + token * (v ? p.v : p.k).sl;
        unsigned char* pages = (v ? p.pages.v : p.pages.k) + to + head * p.pages.sh;
        const u32x4 none = {0u, 0u, 0u, 0u};
        const u32x4 a = ok ? load_chunk(from, c, p.D) : none;
        if constexpr (E4M3) {
            u32x4 codes;
            const uint32_t code = to_e4m3<T>(a, ok ? load_chunk(from, c + 8, p.D) : none, codes);
            if (!ok) continue;
            *reinterpret_cast<u32x4*>(pages + c) = codes;
            if (unit % 2 == 0) (v ? p.pages.vs : p.pages.ks)[scale_to + head * p.pages.scale_sh + unit / 2] = (unsigned char)code;
        } else if (ok) {
            *reinterpret_cast<u32x4*>(pages + 2 * c) = a;
        }
    }
}

// A wave reads one position of a sequence back, K and V of all heads; 32 sequences of 2048 to 4096, 4 heads of 128, e4m3: 70 to 78 us = 5 TB/s.
// k, v: [B, most, Hkv, D], zeros behind a sequence.
template <typename T, bool E4M3>
__global__ __launch_bounds__(kCtxThreads) void paged_read(SeqParams p) {
    const int lane = threadIdx.x & 63;
    const int64_t job = (int64_t)blockIdx.x * kCtxWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (job >= (int64_t)p.B * p.most) return;
    const int b = (int)(job / p.most), position = (int)(job % p.most);
    const int at = p.pages.page_of(position);
    const int page = position < min(p.lengths[b], p.pages.capacity) ? p.pages.table[b * p.pages.table_stride + at] : -1;
    const bool there = (uint32_t)page < (uint32_t)p.pages.pages;
    constexpr int kColumns = E4M3 ? 16 : 8;
    const int per = p.D / kColumns, row = position - at * p.pages.size;
    const int64_t from = p.pages.at(page, row), scale_from = p.pages.scale_at(page, row);
    for (int x = lane; x < 2 * p.Hkv * per; x += 64) {
        const int unit = x % per, hx = x / per, v = hx >= p.Hkv, head = v ? hx - p.Hkv : hx, c = kColumns * unit;
        elem_t* to = (v ? p.v : p.k).head(b, head) + position * (v ? p.v : p.k).sl;
        const unsigned char* pages = (v ? p.pages.v : p.pages.k) + from + head * p.pages.sh;
        u32x4 a = {0u, 0u, 0u, 0u};
        if constexpr (E4M3) {
            u32x4 d = a;
            if (there) {
                const u32x4 codes = *reinterpret_cast<const u32x4*>(pages + c);
                const float scale = scale_of((v ? p.pages.vs : p.pages.ks)[scale_from + head * p.pages.scale_sh + unit / 2]);
                a = from_e4m3_8<T>(codes[0], codes[1], scale), d = from_e4m3_8<T>(codes[2], codes[3], scale);
            }
            *reinterpret_cast<u32x4_any*>(to + c) = a;
            *reinterpret_cast<u32x4_any*>(to + c + 8) = d;
        } else {
            if (there) a = *reinterpret_cast<const u32x4*>(pages + 2 * c);
            *reinterpret_cast<u32x4_any*>(to + c) = a;
        }
    }
}

int paged_copy(const SeqParams& p, bool e4m3, bool fp16, bool write, hipStream_t stream) {
    const int64_t waves = write ? p.T : (int64_t)p.B * p.most;
    const int grid = (int)((waves + kCtxWaves - 1) / kCtxWaves);
    const auto run = [&](auto kernel) { return launch(kernel, grid, 0, stream, p, kCtxThreads); };
    if (!e4m3) return run(write ? paged_write<Bf16, false> : paged_read<Bf16, false>);
    if (fp16) return run(write ? paged_write<Fp16, true> : paged_read<Fp16, true>);
    return run(write ? paged_write<Bf16, true> : paged_read<Bf16, true>);
}

}  // namespace sjvp
