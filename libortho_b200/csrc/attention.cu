// Entry of the attention over a paged cache (attention.cuh): checks, the variant, the workspace.
#include "attention.cuh"

namespace ob {

extern template int launch_attention<__half>(const AttentionArgs &, const AttnPlan &, cudaStream_t);
extern template int launch_attention<__nv_bfloat16>(const AttentionArgs &, const AttnPlan &, cudaStream_t);

static int check_attention(const ortho_b200_paged_attention_desc *d)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->batch < 0 || d->batch > 0x7FFFFFFF || d->q_heads < 1 || d->kv_heads < 1 || d->q_heads > 65535 || d->q_heads % d->kv_heads || d->head_dim < 8 || d->head_dim > 256 || d->head_dim % 8
        || d->rows < 0 || d->pages > 0x7FFFFFFF || d->width < 0 || d->pages < 0 || d->page_size < 1 || d->page_size > 0x7FFFFF00 || d->window < 0 || d->width > 0x7FFFFF00 / d->page_size) return ORTHO_B200_ERR_SHAPE;
    if (d->batch == 0) return ORTHO_B200_OK;
    if (!d->q || !d->k_cache || !d->v_cache || !d->out || !d->lengths || (d->rows && d->width && !d->block_table)) return ORTHO_B200_ERR_NULL;
    if (((uintptr_t)d->q | (uintptr_t)d->k_cache | (uintptr_t)d->v_cache | (uintptr_t)d->out) & 15u) return ORTHO_B200_ERR_ALIGN;
    for (int64_t s : {d->q_token_stride, d->q_head_stride, d->out_token_stride, d->out_head_stride, d->k_page_stride, d->k_slot_stride, d->k_head_stride, d->v_page_stride, d->v_slot_stride, d->v_head_stride})
        if (s % 8) return ORTHO_B200_ERR_ALIGN;
    return ORTHO_B200_OK;
}

template <int DP, int NT> static void take(AttnPlan &p) { p.dp = DP; p.ctas = AttnShape<DP, NT>::kPerSm; p.cluster = AttnShape<DP, NT>::kClusterPerSm; }

constexpr int64_t kJoinUnits = 10;

AttnPlan plan_attention(const ortho_b200_paged_attention_desc &d)
{
    AttnPlan p = {};
    const int64_t heads = d.q_heads / d.kv_heads;
    // The query heads of a key-value head are 8, 16 or (head dims up to 128) 32 columns of one unit, so that the cache is read once; more of
    // them are dealt evenly to several units, which read it again.
    const int64_t most = d.head_dim <= 128 ? 32 : 16;
    p.groups = (int)ceil_div(heads, most);
    p.per_group = (int)ceil_div(heads, p.groups);
    p.groups = (int)ceil_div(heads, p.per_group);
    p.nt = p.per_group <= 8 ? 1 : p.per_group <= 16 ? 2 : 4;
#define OB_CASE(DP)                                                                                   \
    if (!p.dp && d.head_dim <= DP) {                                                                  \
        if (p.nt == 1) take<DP, 1>(p);                                                                \
        else if (p.nt == 2) take<DP, 2>(p);                                                           \
        else take<DP, DP <= 128 ? 4 : 2>(p);                                                          \
    }
    OB_ATTENTION_DIMS(OB_CASE)
#undef OB_CASE
    const int64_t sms = device_sm_count(current_device_index());
    const int64_t keys = d.window > 0 && d.window < d.width * d.page_size ? d.window : d.width * d.page_size;
    const int64_t units = ceil_div(keys, kUnitKeys), items = d.batch * d.kv_heads * p.groups;       // of one item at most; all items
    // An item to a cluster of one to eight CTAs: one launch, nothing passes through memory, but all wait for the longest item.  Or an even cut of all
    // units over all CTAs and join_kernel behind, which takes as long as kJoinUnits units of one CTA more.  The host knows the table's width, not
    // the lengths, so the cut is reckoned with requests of half that on the average.  Measured, clusters / cut, us: 64 + 2 x 8 heads of 128,
    // 1 request of 1000 / 4000 / 8000 keys 5.4 / 10.5 / 19.3, 9.7 / 13.4 / 16.1; 4 of 1000 / 8000 6.6 / 32.0, 12.0 / 30.8; 32 of 100 / 1000
    // 6.7 / 25.5, 10.4 / 32.4, of up to 1000 / 4000 log-spread 18.5 / 64, 14.0 / 22.4; 128 of 100 27.6, 23.8.
    const int64_t room = p.cluster * sms;
    int64_t cluster = items < 1 ? 0 : room / items;
    cluster = cluster >= 8 ? 8 : cluster >= 4 ? 4 : cluster >= 2 ? 2 : p.cluster ? 1 : 0;
    while (cluster > 1 && cluster / 2 >= units) cluster /= 2;
    p.ctas *= (int)sms;
    if (cluster && ceil_div(items * cluster, room) * (ceil_div(units, cluster) + 2) > units * items / (2 * p.ctas) + kJoinUnits) cluster = 0;
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

extern "C" int64_t ortho_b200_paged_attention_workspace_bytes(const ortho_b200_paged_attention_desc *d)
{
    if (check_attention(d) != ORTHO_B200_OK) return -1;
    return d->batch ? plan_attention(*d).bytes : 0;
}

extern "C" int ortho_b200_paged_attention(const ortho_b200_paged_attention_desc *d, void *workspace, int64_t workspace_bytes, void *stream)
{
    int st = check_attention(d);
    if (st || d->batch == 0) return st;
    const AttnPlan p = plan_attention(*d);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255u))) return ORTHO_B200_ERR_WORKSPACE;
    st = check_device();
    if (st) return st;
    AttentionArgs a;
    a.d = *d;
    a.by_page = FastDiv((uint32_t)d->page_size);
    a.scale_log2 = d->scale * 1.4426950408889634f;
    a.per_group = p.per_group; a.groups = p.groups; a.ctas = p.ctas;
    const int64_t rows = 2 * (int64_t)p.ctas * p.nt * 8;
    unsigned char *w = static_cast<unsigned char *>(workspace);
    a.cut = reinterpret_cast<int4 *>(w);
    w += (16 * (int64_t)p.ctas + 255) / 256 * 256;
    a.sums = reinterpret_cast<float2 *>(w);
    w += (8 * rows + 255) / 256 * 256;
    a.part = reinterpret_cast<float *>(w);
    return d->type == ORTHO_B200_TYPE_F16 ? launch_attention<__half>(a, p, (cudaStream_t)stream) : launch_attention<__nv_bfloat16>(a, p, (cudaStream_t)stream);
}
