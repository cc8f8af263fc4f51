// Entry of the attention over a paged cache held in 4 bits (attention_quantised.cuh): checks, the variant, the workspace.
#include "attention_quantised.cuh"

namespace ob {

extern template int launch_attention_quantised<__half>(const QuantisedAttentionArgs &, const AttnPlan &, bool, cudaStream_t);
extern template int launch_attention_quantised<__nv_bfloat16>(const QuantisedAttentionArgs &, const AttnPlan &, bool, cudaStream_t);

static int check_attention_quantised(const ortho_b200_paged_attention_desc *d, const ortho_b200_quantised_cache *c)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    const int st = check_quantised(c);
    if (st) return st;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->batch < 0 || d->batch > 0x7FFFFFFF || d->q_heads < 1 || d->q_heads > 65535 || d->kv_heads != c->kv_heads || d->head_dim != c->head_dim || d->q_heads % c->kv_heads
        || d->rows < 0 || d->width < 0 || d->window < 0 || d->width > 0x7FFFFF00 / c->page_size) return ORTHO_B200_ERR_SHAPE;
    if (d->batch == 0) return ORTHO_B200_OK;
    if (!d->q || !d->out || !d->lengths || (d->rows && d->width && !d->block_table)) return ORTHO_B200_ERR_NULL;
    if (((uintptr_t)d->q | (uintptr_t)d->out) & 15u) return ORTHO_B200_ERR_ALIGN;
    for (int64_t s : {d->q_token_stride, d->q_head_stride, d->out_token_stride, d->out_head_stride})
        if (s % 8) return ORTHO_B200_ERR_ALIGN;
    return expanded(d->batch, d->out_token_stride) || expanded(d->q_heads, d->out_head_stride) ? ORTHO_B200_ERR_SHAPE : ORTHO_B200_OK;
}

template <int DP, int NT, bool GROUPED> static void take(AttnPlan &p)
{
    using Shape = QuantisedShape<DP, NT, GROUPED>;
    p.dp = DP; p.ctas = Shape::kPerSm; p.cluster = Shape::kClusterPerSm;
}

constexpr int64_t kQJoinUnits = 10;

static AttnPlan plan_attention_quantised(const ortho_b200_paged_attention_desc &d, const ortho_b200_quantised_cache &c)
{
    AttnPlan p = {};
    const int64_t heads = d.q_heads / d.kv_heads;
    // As for a 16-bit cache (attention.cu): 8, 16 or, up to 128 elements, 32 query heads of a key-value head meet its keys together
    const int64_t most = d.head_dim <= 128 ? 32 : 16;
    p.groups = (int)ceil_div(heads, most);
    p.per_group = (int)ceil_div(heads, p.groups);
    p.groups = (int)ceil_div(heads, p.per_group);
    p.nt = p.per_group <= 8 ? 1 : p.per_group <= 16 ? 2 : 4;
    const bool grouped = c.groups > 1;
#define OB_CASE(DP)                                                                                                          \
    if (!p.dp && d.head_dim <= DP) {                                                                                         \
        constexpr bool MAY = DP % kQuantGroup == 0 && DP > kQuantGroup;                                                      \
        if (p.nt == 1) { if (grouped) take<DP, 1, MAY>(p); else take<DP, 1, false>(p); }                                     \
        else if (p.nt == 2) { if (grouped) take<DP, 2, MAY>(p); else take<DP, 2, false>(p); }                                \
        else { constexpr int N = DP <= 128 ? 4 : 2; if (grouped) take<DP, N, MAY>(p); else take<DP, N, false>(p); }          \
    }
    OB_QUANTISED_DIMS(OB_CASE)
#undef OB_CASE
    // Clusters or the even cut, as for a 16-bit cache and with the same reckoning.  A unit is 128 keys here instead of 64 and costs about as much (bound by instructions, not bytes), so joining
    // costs as many of them.  Measured, clusters / cut, us: 64 + 2 x 8 heads of 128, 1 request of 1000 / 8000 / 16000 keys 6.7 / 14.2 / 22.8, 10.0 / 17.4 / 21.1; 4 of 1000 / 8000 / 16000
    // 7.9 / 21.3 / 36.5, 12.8 / 23.4 / 35.1; 32 of 100 / 1000 / 4000 8.5 / 22.1 / 66.0, 12.5 / 25.6 / 56.0, of up to 1000 / 4000 log-spread 17.4 / 48.6, 15.6 / 20.7; 128 of 100 23.1, 22.8;
    // 32 + 2 x 2 heads of 256, 1 of 1000 / 8000 10.5 / 25.2, 13.7 / 20.3.
    const int64_t sms = device_sm_count(current_device_index()), width = d.width * c.page_size;
    const int64_t keys = d.window > 0 && d.window < width ? d.window : width;
    const int64_t units = ceil_div(keys, kQUnitKeys), items = d.batch * d.kv_heads * p.groups;      // of one item at most; all items
    const int64_t room = p.cluster * sms;
    int64_t cluster = items < 1 ? 0 : room / items;
    cluster = cluster >= 8 ? 8 : cluster >= 4 ? 4 : cluster >= 2 ? 2 : p.cluster ? 1 : 0;
    while (cluster > 1 && cluster / 2 >= units) cluster /= 2;
    p.ctas *= (int)sms;
    if (cluster && ceil_div(items * cluster, room) * (ceil_div(units, cluster) + 2) > units * items / (2 * p.ctas) + kQJoinUnits) cluster = 0;
    p.cluster = (int)cluster;
    if (cluster) {
        p.ctas = (int)(items * cluster);
        return p;
    }
    // never more CTAs than there can be costs
    if (units < p.ctas && (units + 1) * items < p.ctas) p.ctas = (units + 1) * items < 1 ? 1 : (int)((units + 1) * items);
    const int64_t rows = 2 * (int64_t)p.ctas * p.nt * 8;
    p.bytes = (16 * (int64_t)p.ctas + 255) / 256 * 256 + (8 * rows + 255) / 256 * 256 + 4 * rows * d.head_dim;
    return p;
}

}  // namespace ob

using namespace ob;

extern "C" int64_t ortho_b200_paged_attention_quantised_workspace_bytes(const ortho_b200_paged_attention_desc *d, const ortho_b200_quantised_cache *c)
{
    if (check_attention_quantised(d, c) != ORTHO_B200_OK) return -1;
    return d->batch ? plan_attention_quantised(*d, *c).bytes : 0;
}

extern "C" int ortho_b200_paged_attention_quantised(const ortho_b200_paged_attention_desc *d, const ortho_b200_quantised_cache *c, void *workspace, int64_t workspace_bytes, void *stream)
{
    int st = check_attention_quantised(d, c);
    if (st || d->batch == 0) return st;
    const AttnPlan p = plan_attention_quantised(*d, *c);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255u))) return ORTHO_B200_ERR_WORKSPACE;
    st = check_device();
    if (st) return st;
    QuantisedAttentionArgs args;
    args.c = *c;
    args.wide = c->head_dim % 32 == 0 && (((uintptr_t)c->k | (uintptr_t)c->v) & 15u) == 0;
    for (int64_t s : {c->k_page_stride, c->k_slot_stride, c->k_head_stride, c->v_page_stride, c->v_slot_stride, c->v_head_stride}) args.wide = args.wide && s % 16 == 0;
    // places of a page and a slot in pieces of 16 bytes, and in scales, as 32 bits: the largest of them is the last page's and slot's
    auto number = [&](int64_t page_stride, int64_t slot_stride, int64_t unit, uint32_t &page, uint32_t &slot) {
        if (page_stride < 0 || slot_stride < 0 || page_stride > (1LL << 40) || slot_stride > (1LL << 40) || (c->pages * (page_stride / unit) + c->page_size * (slot_stride / unit)) >= (1LL << 32)) args.wide = 0;
        page = (uint32_t)(page_stride / unit);
        slot = (uint32_t)(slot_stride / unit);
    };
    number(c->k_page_stride, c->k_slot_stride, 16, args.k_page, args.k_slot);
    number(c->v_page_stride, c->v_slot_stride, 16, args.v_page, args.v_slot);
    number(c->ks_page_stride, c->ks_slot_stride, 1, args.ks_page, args.ks_slot);
    number(c->vs_page_stride, c->vs_slot_stride, 1, args.vs_page, args.vs_slot);
    AttentionArgs &a = args.a;
    a.d = *d;
    a.d.pages = c->pages;
    a.d.page_size = c->page_size;
    if (c->pages == 0) a.d.width = 0;            // nothing is cached: no row has a key
    a.by_page = FastDiv((uint32_t)c->page_size);
    a.scale_log2 = d->scale * 1.4426950408889634f;
    a.per_group = p.per_group; a.groups = p.groups; a.ctas = p.ctas;
    const int64_t rows = 2 * (int64_t)p.ctas * p.nt * 8;
    unsigned char *w = static_cast<unsigned char *>(workspace);
    a.cut = reinterpret_cast<int4 *>(w);
    w += (16 * (int64_t)p.ctas + 255) / 256 * 256;
    a.sums = reinterpret_cast<float2 *>(w);
    w += (8 * rows + 255) / 256 * 256;
    a.part = reinterpret_cast<float *>(w);
    const bool grouped = c->groups > 1;
    return d->type == ORTHO_B200_TYPE_F16 ? launch_attention_quantised<__half>(args, p, grouped, (cudaStream_t)stream)
                                          : launch_attention_quantised<__nv_bfloat16>(args, p, grouped, (cudaStream_t)stream);
}
