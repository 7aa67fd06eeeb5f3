// C ABI of the attention on keys of another length / with a relative position bias (sjvp_ctx_fwd, sjvp_ctx_bwd): checks, how
// the work is split, and the launches.
#include <climits>
#include <cmath>
#include <type_traits>

#include "sjvp_ctx_launch.hpp"

namespace sjvp {

// Adds up the bucket sums of the workgroups of a head: 16 threads to a bucket, each over every 16th workgroup, in a fixed order.
__global__ __launch_bounds__(256) void ctx_table_sum(CtxParams p) {
    __shared__ float sums[16][17];
    const int nb = p.both ? 2 * p.buckets : p.buckets, per = (nb + 15) / 16;
    const int head = blockIdx.x / per, col = threadIdx.x & 15, slice = threadIdx.x >> 4, bucket = (blockIdx.x % per) * 16 + col;
    const int64_t parts = (int64_t)p.B * p.blocks * p.splits;
    float sum = 0.0f;
    if (bucket < nb)
        for (int64_t i = slice; i < parts; i += 16) sum += p.tpart[((int64_t)head * parts + i) * nb + bucket];
    sums[slice][col] = sum;
    workgroup_barrier();
    if (slice == 0 && bucket < nb) {
        sum = 0.0f;
        for (int i = 0; i < 16; ++i) sum += sums[i][col];
        const int64_t at = bucket * p.dtsb + head * p.dtsh;
        if (p.table_type == SJVP_FP32) reinterpret_cast<float*>(p.dtable)[at] = sum;
        else reinterpret_cast<elem_t*>(p.dtable)[at] = (elem_t)(p.table_type == SJVP_BF16 ? Bf16::pack2(sum, 0.0f) : Fp16::pack2(sum, 0.0f));
    }
}

namespace {

constexpr int kMaxSplits = 64;
constexpr int kLds = 160 * 1024;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits of a looped axis of `steps` steps for a launch of `groups` workgroups: up to one workgroup to a compute unit, each with `least`
// steps or more.
int splits_for(int64_t groups, int64_t steps, int64_t least) {
    const int64_t wanted = compute_units() / groups;
    return (int)std::max<int64_t>(1, std::min<int64_t>({wanted, steps / least, kMaxSplits}));
}

}  // namespace

// Times of the rules below in microseconds, D = 64 unless said, (B,Hq,Lq,Lk) bf16; `rel`: with a bias.  They ask for compute units and tiles
// alone: of D <= 32 and D > 64 the backward's were measured at the entries given, not over a range.
//
// Few rows (ctx_fwd_few) where the rows of a key head fit one block, and where blocks of 128 rows would leave half of the compute
// units idle: (2,8,512,1024) rel 15.2 / 31.4 by blocks of 128, (2,16,200,2000) D=128 28 / 65, (4,16,256,1024) 18.5 / 20.6; beyond
// that (8,16,256,256) rel 21.6 / 14.4, (16,12,128,128) rel 11.8 / 10.2.
//   waves: eight share the filling of a bias row for many keys, (2,8,512,1024) rel 11.5 / 12.7 with four; otherwise four, which end sooner:
//     (64,12,1,400) 17.8 / 21.1 with eight, (4,12,256,256) rel 9.6 / 10.4, (2,16,4,16385) D=128 in groups of eight 15.2 / 16.3.
//   packed heads read their keys once: (64,16,1,2048) D=128 in groups of four 45 / 160 one by one.
//   splits: of 256 keys or more, since joining them is a launch of 4 us: (8,16,4,2000) D=128 in groups of eight 13.2 / 22.7 unsplit,
//     (1,12,1,2000) rel 12.1 / 18.1; none up to 1024 keys at D = 64: (1,8,300,1000) 10.7 / 11.7 split, (1,12,1,600) 8.1 / 8.9.
CtxPlan ctx_plan_fwd(const CtxParams& p) {
    CtxPlan plan;
    const int HD = ctx_padded(p.D), bias = p.table ? 4 * ctx_entries(p) : 0;
    const int64_t many = (int64_t)p.B * p.Hq * ceil_div(p.Lq, kCtxOwned);
    plan.few = (int64_t)p.G * p.Lq <= 32 || 2 * many <= compute_units();
    if (!plan.few) {
        plan.blocks = (int)ceil_div(p.Lq, kCtxOwned);
        plan.units = (int64_t)p.B * p.Hkv;
        plan.inner = (int64_t)p.G * plan.blocks;
        plan.dma = ctx_dma(p, p.k, p.v);
        plan.smem = ctx_tiles_bytes(HD, plan.dma) + bias;
        return plan;
    }
    const int heads = p.Lq < 32 ? std::min(p.G, 31 / p.Lq + 2) : 1;  // that a block of 32 rows can touch
    const auto sums = [&](int waves) { return waves * 32 * (HD + 4 + 2) * 4; };
    plan.waves = p.table && p.Lk >= 1024 && sums(8) + heads * bias <= kLds ? 8 : 4;
    plan.packed = p.Lq < 32 && sums(plan.waves) + heads * bias <= kLds ? p.G : 1;
    plan.smem = sums(plan.waves) + (plan.packed > 1 ? heads : 1) * bias;
    plan.blocks = (int)ceil_div((int64_t)plan.packed * p.Lq, 32);
    plan.units = (int64_t)p.B * p.Hkv * (p.G / plan.packed);
    plan.splits = (int64_t)p.Lk * HD <= 1024 * 64 ? 1 : splits_for(plan.units * plan.blocks, p.Lk, 256);
    plan.inner = (int64_t)plan.blocks * plan.splits;
    return plan;
}

// The backward pair splits its looped axes from ten tiles on while compute units are idle: the launch that adds up costs 4 us and the
// partial sums their traffic.  (4,8,512,512) rel whole 42, in tiles of four 50; (2,8,512,1024) rel 44 / 49; the other way (8,8,300,300) D=36
// rel in groups of two 52 in tiles of five, 58 whole, (1,8,300,300) D=128 rel in groups of two 54 / 64.
CtxPlan ctx_plan_row(const CtxParams& p) {
    CtxPlan plan;
    plan.blocks = (int)ceil_div(p.Lq, kCtxOwned);
    plan.units = (int64_t)p.B * p.Hkv;
    plan.splits = splits_for((int64_t)p.B * p.Hq * plan.blocks, ceil_div(p.Lk, kCtxTile), 5);
    plan.inner = (int64_t)p.G * plan.blocks * plan.splits;
    plan.dma = ctx_dma(p, p.k, p.v);
    plan.smem = ctx_tiles_bytes(ctx_padded(p.D), plan.dma) + (p.table ? 4 * ctx_entries(p) * (1 + kCtxWaves) : 0);
    return plan;
}

CtxPlan ctx_plan_col(const CtxParams& p) {
    CtxPlan plan;
    plan.blocks = (int)ceil_div(p.Lk, kCtxOwned);
    plan.units = (int64_t)p.B * p.Hkv;
    plan.splits = splits_for(plan.units * plan.blocks, p.G * ceil_div(p.Lq, kCtxTile), 5);
    plan.inner = (int64_t)plan.blocks * plan.splits;
    plan.dma = ctx_dma(p, p.q, p.g);
    plan.smem = ctx_tiles_bytes(ctx_padded(p.D), plan.dma) + 4 * kCtxStats + (p.table ? 4 * ctx_entries(p) : 0);
    return plan;
}

// The single backward launch, against the pair.  Its workgroup walks all rows of its heads, so that the pair spreads few of them over
// more compute units, unless the walk is short.  One workgroup of eight waves fills a compute unit: a last round that leaves many idle costs a
// whole one.
//   up to three tiles: 8 heads of 64 rows on 100 keys 8.6 / 13.0 by the pair, of 192 rows 15.7 / 16.7 (rel 26 / 25), of 256 rows rel 31 / 27;
//     (8,12,128,128) 13.0 / 15.5, (11,16,100,200) rel 25 / 31, (8,16,128,256) 17 / 18.5
//   four waves (up to 128 keys): (24,16,512,128) 50 / 60, (64,12,128,128) rel 50 / 59; few workgroups (4,16,256,128) 20.4 / 18.8, (4,16,1024,128) 65 / 36
//   eight waves: (10,16,256,200) 27 / 30.5, (16,16,256,256) 30 / 34, (28,16,300,256) 65 / 70, (64,12,1024,256) 245 / 299; the other way
//     (8,16,256,256) rel 37 / 34, (24,16,256,256) 52 / 47, (40,16,256,256) 78 / 73, (32,12,1024,256) 158 / 140
bool ctx_plan_one(const CtxParams& p, CtxPlan& plan) {
    if (ctx_padded(p.D) != 64 || p.Lk > 256 || !p.dk.ptr) return false;
    plan.waves = p.Lk > 128 ? 8 : 4;
    plan.units = (int64_t)p.B * p.Hkv;
    plan.dma = ctx_dma(p, p.q, p.g) && ctx_aligned(p.k);
    const int tile = kCtxTile * (64 + (plan.dma ? 0 : 8)) * 2;
    const int ds = plan.waves / 2 * kCtxTile * 72 * 2;
    plan.smem = (plan.waves / 2 + 4) * tile + ds + 4 * kCtxStats + (p.table ? 4 * (ctx_entries(p) * (1 + plan.waves) + 28) : 0);
    if (plan.smem > kLds) return false;
    plan.packed = plan.waves == 8 && plan.smem + ds <= kLds ? 2 : 1;
    plan.smem += (plan.packed - 1) * ds;
    const int64_t units = plan.units, cu = compute_units(), rounds = ceil_div(units, cu);
    if (rounds == 1 && p.G * ceil_div(p.Lq, kCtxTile) <= 3) return true;
    if (plan.waves == 4) return 2 * units >= cu;
    return rounds == 1 ? 5 * units >= 3 * cu : 7 * units >= 6 * rounds * cu;
}

namespace {

int ctx_params(const sjvp_ctx* t, CtxParams& p) {
    if (!t) return SJVP_ERR_NULL;
    if (t->B < 1 || t->Hq < 1 || t->Hkv < 1 || t->Lq < 1 || t->Lk < 1 || t->Hq % t->Hkv || t->Lq > kCtxMost || t->Lk > kCtxMost ||
        t->query_start0 > kCtxMost || t->query_start0 < -kCtxMost)
        return SJVP_ERR_SHAPE;
    if (t->D < 16 || t->D > 128) return SJVP_ERR_HEAD_DIM;
    if (!(t->scale >= 0.0f) || !std::isfinite(t->scale)) return SJVP_ERR_SCALE;
    CtxView* views[SJVP_C_COUNT] = {&p.q, &p.k, &p.v, &p.o, &p.rest, &p.g, &p.dq, &p.dk, &p.dv};
    const void* ptrs[SJVP_C_COUNT] = {t->q, t->k, t->v, t->o, t->o_rest, t->dO, t->dq, t->dk, t->dv};
    for (int i = 0; i < SJVP_C_COUNT; ++i)
        *views[i] = {static_cast<elem_t*>(const_cast<void*>(ptrs[i])), t->strides[3 * i], t->strides[3 * i + 1], t->strides[3 * i + 2]};
    for (CtxView* v : {&p.q, &p.g})
        if (t->Lq == 1) v->sl = t->D;  // (one row: no stride)
    for (CtxView* v : {&p.k, &p.v})
        if (t->Lk == 1) v->sl = t->D;
    for (const CtxView* v : {&p.q, &p.k, &p.v, &p.g})
        if (v->ptr && (v->sl < 0 || v->sl >= 1 << 24)) return SJVP_ERR_SHAPE;
    p.lse = t->lse;
    p.klen = t->key_lengths, p.qlen = t->query_lengths, p.start = t->query_start, p.start0 = t->query_start0;
    p.B = t->B, p.Hq = t->Hq, p.Hkv = t->Hkv, p.G = t->Hq / t->Hkv, p.Lq = t->Lq, p.Lk = t->Lk, p.D = t->D;
    p.scale = t->scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(t->D)) : t->scale;
    p.c = p.scale * kLog2e;
    p.table = t->table, p.dtable = t->dtable, p.table_type = t->table_dtype;
    p.tsb = t->table_stride[0], p.tsh = t->table_stride[1], p.dtsb = t->dtable_stride[0], p.dtsh = t->dtable_stride[1];
    p.both = t->bidirectional != 0, p.causal = t->causal != 0;
    if (!t->table) return p.causal || t->dtable ? SJVP_ERR_BUCKETS : SJVP_OK;
    if (t->table_dtype != SJVP_FP32 && t->table_dtype != SJVP_BF16 && t->table_dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->bucket_first) return SJVP_ERR_NULL;
    if (t->buckets < 1 || t->buckets > kCtxBuckets || t->bucket_first[0] != 0) return SJVP_ERR_BUCKETS;
    p.buckets = t->buckets;
    for (int i = 0; i < t->buckets; ++i) {
        if (t->bucket_first[i] > SJVP_CTX_MAX_DISTANCE || (i && t->bucket_first[i] < t->bucket_first[i - 1])) return SJVP_ERR_BUCKETS;
        p.first[i] = static_cast<uint16_t>(t->bucket_first[i]);
    }
    p.far = std::max(1, t->bucket_first[t->buckets - 1]);
    return SJVP_OK;
}

// The plans of a call, and where its scratch lies in the workspace (in floats).
struct CtxLayout {
    CtxPlan fwd, row, col, one;
    bool single = false;  // backward by ctx_bwd_one
    size_t folded = 0, tpart = 0, stat = 0, part = 0, total = 0;
};

CtxLayout ctx_layout(const CtxParams& p, bool backward) {
    CtxLayout l;
    const size_t HD = ctx_padded(p.D), q_rows = (size_t)p.B * p.Hq * p.Lq, k_rows = (size_t)p.B * p.Hkv * p.Lk;
    const auto take = [&](size_t floats) {
        const size_t at = l.total;
        l.total += (floats + 3) / 4 * 4;
        return at;
    };
    if (!backward) {
        l.fwd = ctx_plan_fwd(p);
        if (l.fwd.splits > 1) {
            l.stat = take(2 * l.fwd.splits * q_rows);
            l.part = take(l.fwd.splits * q_rows * HD);
        }
        return l;
    }
    l.single = ctx_plan_one(p, l.one);
    if (l.single) {
        if (p.dtable) l.tpart = take((size_t)p.Hq * p.B * (p.both ? 2 : 1) * p.buckets);
        return l;
    }
    l.row = ctx_plan_row(p);
    l.col = ctx_plan_col(p);
    l.folded = take(3 * q_rows);
    if (p.dtable) l.tpart = take((size_t)p.Hq * p.B * l.row.blocks * l.row.splits * (p.both ? 2 : 1) * p.buckets);
    // (the row-owned launch's sums are used up before the column-owned one writes its own)
    const size_t row = l.row.splits > 1 ? l.row.splits * q_rows * HD : 0, col = l.col.splits > 1 ? 2 * l.col.splits * k_rows * HD : 0;
    l.part = take(std::max(row, col));
    return l;
}

// A launch holds fewer than 2^32 threads.
bool ctx_fits(const CtxPlan& plan) {
    return std::max(plan.units, plan.inner) <= INT_MAX && ctx_grid(plan.units, plan.inner) <= UINT32_MAX / (64 * plan.waves);
}

int ctx_workspace(const sjvp_ctx* t, const CtxLayout& l, float*& ws) {
    ws = static_cast<float*>(t->workspace);
    return l.total == 0 || (ws && t->workspace_bytes >= 4 * l.total && reinterpret_cast<uintptr_t>(ws) % 16 == 0) ? SJVP_OK : SJVP_ERR_WORKSPACE;
}

}  // namespace
}  // namespace sjvp

extern "C" {

using namespace sjvp;

size_t sjvp_ctx_workspace_bytes(const sjvp_ctx* t, int backward) {
    CtxParams p{};
    if (ctx_params(t, p) != SJVP_OK) return 0;
    return 4 * ctx_layout(p, backward != 0).total;
}

int sjvp_ctx_fwd(const sjvp_ctx* t, int dtype, void* stream) {
    CtxParams p{};
    const int rc = ctx_params(t, p);
    if (rc != SJVP_OK) return rc;
    if (dtype != SJVP_BF16 && dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->q || !t->k || !t->v || !t->o) return SJVP_ERR_NULL;
    const CtxLayout l = ctx_layout(p, false);
    if (!ctx_fits(l.fwd)) return SJVP_ERR_SHAPE;
    float* ws;
    if (ctx_workspace(t, l, ws) != SJVP_OK) return SJVP_ERR_WORKSPACE;
    p.stat = ws + l.stat, p.part = ws + l.part;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SJVP_BF16 ? ctx_forward<Bf16>(p, l.fwd, s) : ctx_forward<Fp16>(p, l.fwd, s);
}

int sjvp_ctx_bwd(const sjvp_ctx* t, int dtype, void* stream) {
    CtxParams p{};
    int rc = ctx_params(t, p);
    if (rc != SJVP_OK) return rc;
    if (dtype != SJVP_BF16 && dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->q || !t->k || !t->v || !t->o || !t->dO || !t->dq || !t->dk != !t->dv || !t->lse) return SJVP_ERR_NULL;
    CtxLayout l = ctx_layout(p, true);
    const int64_t per = ((p.both ? 2 : 1) * p.buckets + 15) / 16;  // workgroups of ctx_table_sum to a head
    if (!ctx_fits(l.row) || !ctx_fits(l.col) || !ctx_fits(l.one) || p.Hq * per > UINT32_MAX / 256) return SJVP_ERR_SHAPE;
    float* ws;
    if (ctx_workspace(t, l, ws) != SJVP_OK) return SJVP_ERR_WORKSPACE;
    p.folded = ws + l.folded, p.part = ws + l.part, p.tpart = p.dtable ? ws + l.tpart : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const auto run = [&](const CtxPlan& plan, bool row) {
        return dtype == SJVP_BF16 ? ctx_backward<Bf16>(p, plan, row, s) : ctx_backward<Fp16>(p, plan, row, s);
    };
    if (l.single) {
        rc = dtype == SJVP_BF16 ? ctx_backward_one<Bf16>(p, l.one, s) : ctx_backward_one<Fp16>(p, l.one, s);
        l.row.blocks = l.row.splits = 1;
    } else {
        rc = run(l.row, true);
        if (rc == SJVP_OK && t->dk) rc = run(l.col, false);
    }
    if (rc != SJVP_OK || !p.dtable) return rc;
    p.blocks = l.row.blocks, p.splits = l.row.splits;
    return launch(ctx_table_sum, (int)(p.Hq * per), 0, s, p, 256);
}

}  // extern "C"
