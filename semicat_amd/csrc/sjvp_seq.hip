// C ABI of the attention over packed sequences and over a paged cache: checks, how the work is split, and the launches.
#include <climits>
#include <cmath>

#include "sjvp_seq_launch.hpp"

namespace sjvp {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// a launch has fewer than 2^32 threads
int seq_grid(int64_t blocks, int threads) { return blocks > UINT32_MAX / threads ? SJVP_ERR_SHAPE : SJVP_OK; }

bool strides_ok(const CtxView& v, int rows) { return rows <= 1 || (v.sl >= 0 && v.sl < 1 << 24); }

// what the calls have in common
int seq_common(SeqParams& p, int B, int T, int Hq, int Hkv, int D, float scale) {
    if (B < 1 || T < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || B > kCtxMost || T > kCtxMost || (int64_t)T * Hq > INT_MAX) return SJVP_ERR_SHAPE;
    if (D < 16 || D > 128) return SJVP_ERR_HEAD_DIM;
    if (!(scale >= 0.0f) || !std::isfinite(scale)) return SJVP_ERR_SCALE;
    p.B = B, p.T = T, p.Hq = Hq, p.Hkv = Hkv, p.G = Hq / Hkv, p.D = D;
    p.scale = scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(D)) : scale;
    p.c = p.scale * kLog2e;
    return SJVP_OK;
}

// The backward of whole sequences: the column-owned launch is split over the heads that share a key head, as far as four workgroups to a compute unit
// (four sequences of 1024 to 2048 tokens, Hq=32 Hkv=4 D=128, forward and backward: 476 us; one 677, two 489, eight 494; of 1500 to 6000, Hq=16: 1244,
// 1364, 1358 and 1286).
struct PackedPlan {
    int splits = 1;
    size_t part = 0, total = 0;  // floats
};

PackedPlan packed_plan(const SeqParams& p) {
    PackedPlan plan;
    const int64_t blocks = (p.T / kCtxOwned + 1) * (int64_t)p.Hkv;
    plan.splits = (int)std::max<int64_t>(1, std::min<int64_t>(4 * (int64_t)compute_units() / blocks, p.G));
    plan.part = (3 * (size_t)p.Hq * p.T + 3) / 4 * 4;
    plan.total = plan.part + (plan.splits > 1 ? 2 * (size_t)plan.splits * p.Hkv * p.T * ctx_padded(p.D) : 0);
    return plan;
}

int packed_params(const sjvp_packed* t, SeqParams& p) {
    if (!t) return SJVP_ERR_NULL;
    const int rc = seq_common(p, t->B, t->T, t->Hq, t->Hkv, t->D, t->scale);
    if (rc != SJVP_OK) return rc;
    CtxView* views[SJVP_S_COUNT] = {&p.q, &p.k, &p.v, &p.o, &p.g, &p.dq, &p.dk, &p.dv};
    const void* ptrs[SJVP_S_COUNT] = {t->q, t->k, t->v, t->o, t->dO, t->dq, t->dk, t->dv};
    for (int i = 0; i < SJVP_S_COUNT; ++i) *views[i] = {static_cast<elem_t*>(const_cast<void*>(ptrs[i])), 0, t->strides[2 * i], t->strides[2 * i + 1]};
    for (CtxView* v : {&p.q, &p.k, &p.v, &p.g}) {
        if (v->ptr && !strides_ok(*v, t->T)) return SJVP_ERR_SHAPE;
        if (t->T == 1) v->sl = t->D;  // (one row: no stride)
    }
    p.lse = t->lse, p.offsets = t->offsets, p.causal = t->causal != 0;
    if (seq_grid(seq_slots(p, p.G, kCtxOwned) * p.Hkv, kCtxThreads) != SJVP_OK) return SJVP_ERR_SHAPE;
    return seq_grid(seq_slots(p, 1, kCtxOwned) * p.Hkv * packed_plan(p).splits, 2 * kCtxThreads);
}

int paged_params(const sjvp_paged* t, SeqParams& p, int T) {
    if (!t) return SJVP_ERR_NULL;
    const int rc = seq_common(p, t->B, T, t->Hq, t->Hkv, t->D, t->scale);
    if (rc != SJVP_OK) return rc;
    const bool e4m3 = t->k_scales || t->v_scales;
    if (t->pages < 1 || t->page_size < 1 || t->page_size > kCtxMost || t->table_pages < 1 || t->D % (e4m3 ? 16 : 8)) return SJVP_ERR_PAGES;
    if (!t->k_pages || !t->v_pages || !t->tables || !t->lengths || !t->k_scales != !t->v_scales) return SJVP_ERR_NULL;
    for (int i = 0; i < 3; ++i)
        if (t->page_strides[i] % 16 || t->page_strides[i] < 0) return SJVP_ERR_PAGES;
    for (int i : {0, 2, 3, 5})
        if (t->page_strides[i] < 0 || t->page_strides[i] > UINT32_MAX) return SJVP_ERR_PAGES;
    if (reinterpret_cast<uintptr_t>(t->k_pages) % 16 || reinterpret_cast<uintptr_t>(t->v_pages) % 16) return SJVP_ERR_PAGES;
    CtxView* views[SJVP_P_COUNT] = {&p.q, &p.o, &p.k, &p.v};
    const void* ptrs[SJVP_P_COUNT] = {t->q, t->o, t->k, t->v};
    for (int i = 0; i < SJVP_P_COUNT; ++i)
        *views[i] = {static_cast<elem_t*>(const_cast<void*>(ptrs[i])), t->strides[3 * i + 2], t->strides[3 * i], t->strides[3 * i + 1]};
    p.lengths = t->lengths, p.offsets = t->offsets, p.causal = 1;
    SeqPages& g = p.pages;
    g.k = static_cast<unsigned char*>(t->k_pages), g.v = static_cast<unsigned char*>(t->v_pages);
    g.ks = static_cast<unsigned char*>(t->k_scales), g.vs = static_cast<unsigned char*>(t->v_scales);
    g.sp = (uint32_t)t->page_strides[0], g.sh = t->page_strides[1], g.sr = (uint32_t)t->page_strides[2];
    g.scale_sp = (uint32_t)t->page_strides[3], g.scale_sh = t->page_strides[4], g.scale_sr = (uint32_t)t->page_strides[5];
    g.table = t->tables, g.table_stride = t->table_stride;
    g.pages = t->pages, g.size = t->page_size;
    g.capacity = (int)std::min<int64_t>((int64_t)t->table_pages * t->page_size, kCtxMost);
    const int groups = (t->D + 31) / 32;
    g.scale_words = (((uintptr_t)g.ks | (uintptr_t)g.vs | (uintptr_t)g.scale_sp | (uintptr_t)g.scale_sh | (uintptr_t)g.scale_sr) & (groups - 1)) == 0;
    g.shift = 0;
    while ((1u << g.shift) < (uint32_t)g.size) ++g.shift;
    g.magic = (uint32_t)(((uint64_t(1) << (31 + g.shift)) + g.size - 1) / g.size);
    return SJVP_OK;
}

PagedPlan paged_plan(const SeqParams& p) {
    PagedPlan plan;
    const int64_t rows = (int64_t)p.T * p.G, cu = compute_units(), keys = p.pages.capacity;
    const auto take = [&](int64_t floats) {
        const size_t at = plan.total;
        plan.total += (size_t)(floats + 3) / 4 * 4;
        return at;
    };
    const auto scratch = [&](PagedPart& part, int64_t places) {
        if (part.splits <= 1) return;
        part.stat = take(2 * part.splits * places);
        part.part = take(part.splits * places * ctx_padded(p.D));
        part.used = take(places);
    };
    const auto splits = [](int64_t wanted, int64_t most, int64_t limit) { return (int)std::max<int64_t>(1, std::min<int64_t>({wanted, most, limit})); };
    const int64_t many = ceil_div(rows, kCtxOwned) * p.Hkv;
    // seq_fwd's blocks of 128 rows, where the sequences have 128 rows on average (H=28 G=4 D=64 e4m3, 37 sequences of 0 to 32 new tokens on up to 2490:
    // 86 us with it, 41 without; 46 of up to 125, G=8: 26 and 50) and are many enough, which for a long cache is fewer blocks, each split over its keys
    // (16 heads, 512 tokens on 32768: 190 us, 276 by seq_few; five sequences of 463 tokens, 95 blocks: 23 and 15).  Sequences of few rows
    // have seq_few beside it unless 256 rows on average make such unlikely (one decodes while another's prompt is read).
    plan.has_many = rows >= 128 * (int64_t)p.B && p.T > p.B && (keys < 1024 ? 2 : 8) * many > cu;
    plan.has_few = !plan.has_many || rows < 256 * (int64_t)p.B;
    if (plan.has_few) {
        // Splits of 256 keys or more, 512 of 8 bits, which take half of the bytes (a token each of 11 sequences of 604, 17 heads: 16.3 us at 256, 12.9; of
        // 21600 tokens of 16 bits, two heads: 15.3 and 17.8 at 384): as many as give eight workgroups to a compute unit (57 sequences of up to 20
        // tokens on up to 10334, D=64: 54 us, 62 with half as many).  Below 768 keys the join costs more (16 tokens on 600, 8 heads: 14.9 us split, 12.3).
        plan.few.split_tiles = p.pages.ks ? 16 : 8;
        plan.few.splits = keys < 768 ? 1 : splits(8 * cu / ((p.B + rows / 32) * p.Hkv), keys / (32 * plan.few.split_tiles), 128);
        scratch(plan.few, p.Hkv * (plan.has_many ? (int64_t)(p.B + 2) * kSeqFew : rows));
    }
    if (plan.has_many) {
        // Splits of 2048 keys (1024: eight prompts of 512 tokens on up to 8192, 212 us in place of 187), of 512 where there are few blocks.
        plan.many.split_tiles = 2 * many > cu ? 32 : 8;
        plan.many.splits = splits(8 * cu / many, keys / (kCtxTile * plan.many.split_tiles), 16);
        scratch(plan.many, p.Hkv * rows);
    }
    return plan;
}

// (splits are made of launches of few blocks alone, so that those of one split are the most)
int attention_params(const sjvp_paged* t, SeqParams& p) {
    const int rc = paged_params(t, p, t->T);
    return rc != SJVP_OK ? rc : seq_grid(seq_slots(p, p.G, 16 * seq_sets(p)) * p.Hkv, kCtxThreads);
}

int seq_workspace(void* ws, size_t bytes, size_t floats) {
    return floats == 0 || (ws && bytes >= 4 * floats && reinterpret_cast<uintptr_t>(ws) % 16 == 0) ? SJVP_OK : SJVP_ERR_WORKSPACE;
}

}  // namespace
}  // namespace sjvp

extern "C" {

using namespace sjvp;

size_t sjvp_packed_workspace_bytes(const sjvp_packed* t, int backward) {
    SeqParams p{};
    return backward && packed_params(t, p) == SJVP_OK ? 4 * packed_plan(p).total : 0;
}

int sjvp_packed_fwd(const sjvp_packed* t, int dtype, void* stream) {
    SeqParams p{};
    const int rc = packed_params(t, p);
    if (rc != SJVP_OK) return rc;
    if (dtype != SJVP_BF16 && dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->q || !t->k || !t->v || !t->o || !t->offsets) return SJVP_ERR_NULL;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SJVP_BF16 ? seq_packed_fwd<Bf16>(p, s) : seq_packed_fwd<Fp16>(p, s);
}

int sjvp_packed_bwd(const sjvp_packed* t, int dtype, void* stream) {
    SeqParams p{};
    const int rc = packed_params(t, p);
    if (rc != SJVP_OK) return rc;
    if (dtype != SJVP_BF16 && dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->q || !t->k || !t->v || !t->o || !t->dO || !t->dq || !t->dk != !t->dv || !t->lse || !t->offsets) return SJVP_ERR_NULL;
    const PackedPlan plan = packed_plan(p);
    if (seq_workspace(t->workspace, t->workspace_bytes, plan.total) != SJVP_OK) return SJVP_ERR_WORKSPACE;
    p.splits = plan.splits, p.folded = static_cast<float*>(t->workspace), p.part = p.folded + plan.part;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SJVP_BF16 ? seq_packed_bwd<Bf16>(p, s) : seq_packed_bwd<Fp16>(p, s);
}

size_t sjvp_paged_workspace_bytes(const sjvp_paged* t) {
    SeqParams p{};
    return t && attention_params(t, p) == SJVP_OK ? 4 * paged_plan(p).total : 0;
}

int sjvp_paged_write(const sjvp_paged* t, int dtype, void* stream) {
    SeqParams p{};
    const int rc = t ? paged_params(t, p, t->T) : SJVP_ERR_NULL;
    if (rc != SJVP_OK) return rc;
    if (dtype != SJVP_BF16 && dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->k || !t->v || (!t->offsets && t->T != t->B)) return SJVP_ERR_NULL;
    if (seq_grid(t->T, 64) != SJVP_OK) return SJVP_ERR_SHAPE;  // (a wave to a token)
    return paged_copy(p, p.pages.ks, dtype == SJVP_FP16, true, static_cast<hipStream_t>(stream));
}

int sjvp_paged_read(const sjvp_paged* t, int dtype, void* stream) {
    SeqParams p{};
    const int rc = paged_params(t, p, 1);
    if (rc != SJVP_OK) return rc;
    if (dtype != SJVP_BF16 && dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->k || !t->v) return SJVP_ERR_NULL;
    if (t->size < 1 || t->size > kCtxMost || seq_grid((int64_t)t->B * t->size, 64) != SJVP_OK) return SJVP_ERR_SHAPE;
    p.most = t->size;
    return paged_copy(p, p.pages.ks, dtype == SJVP_FP16, false, static_cast<hipStream_t>(stream));
}

int sjvp_paged_attention(const sjvp_paged* t, int dtype, void* stream) {
    SeqParams p{};
    const int rc = t ? attention_params(t, p) : SJVP_ERR_NULL;
    if (rc != SJVP_OK) return rc;
    if (dtype != SJVP_BF16 && dtype != SJVP_FP16) return SJVP_ERR_DTYPE;
    if (!t->q || !t->o || (!t->offsets && t->T != t->B)) return SJVP_ERR_NULL;
    const PagedPlan plan = paged_plan(p);
    if (seq_workspace(t->workspace, t->workspace_bytes, plan.total) != SJVP_OK) return SJVP_ERR_WORKSPACE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(t->workspace);
    return dtype == SJVP_BF16 ? seq_paged<Bf16>(p, plan, ws, p.pages.ks, s) : seq_paged<Fp16>(p, plan, ws, p.pages.ks, s);
}

}  // extern "C"
