// The paged cache held in 4 bits (include/ortho_b200.h has the format): the checks of its record.
#pragma once

#include "launch.cuh"

namespace ob {

constexpr int kQuantGroup = 64;                  // elements of a group that is not a whole head

inline int check_quantised(const ortho_b200_quantised_cache *c)
{
    if (!c) return ORTHO_B200_ERR_NULL;
    if (c->pages < 0 || c->pages > 0x7FFFFFFF || c->page_size < 1 || c->page_size > 0x7FFFFF00 || c->kv_heads < 1 || c->kv_heads > 65535 || c->head_dim < 8 || c->head_dim > 256
        || c->head_dim % 8 || c->groups < 1 || (c->groups > 1 && c->groups * kQuantGroup != c->head_dim)) return ORTHO_B200_ERR_SHAPE;
    if (c->pages && (!c->k || !c->v || !c->k_scales || !c->v_scales)) return ORTHO_B200_ERR_NULL;
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 3u) return ORTHO_B200_ERR_ALIGN;
    for (int64_t s : {c->k_page_stride, c->k_slot_stride, c->k_head_stride, c->v_page_stride, c->v_slot_stride, c->v_head_stride})
        if (s % 4) return ORTHO_B200_ERR_ALIGN;
    return ORTHO_B200_OK;
}

// Entries of a dimension that is written would lie in one place
inline bool expanded(int64_t entries, int64_t stride) { return entries > 1 && stride == 0; }

// A cache that is written: no two tokens or heads in one place, keys apart from values
inline int check_written(const ortho_b200_quantised_cache &c)
{
    if (c.pages == 0) return ORTHO_B200_OK;
    if (c.k == c.v || c.k_scales == c.v_scales) return ORTHO_B200_ERR_SHAPE;
    for (int64_t s : {c.k_page_stride, c.v_page_stride, c.ks_page_stride, c.vs_page_stride}) if (expanded(c.pages, s)) return ORTHO_B200_ERR_SHAPE;
    for (int64_t s : {c.k_slot_stride, c.v_slot_stride, c.ks_slot_stride, c.vs_slot_stride}) if (expanded(c.page_size, s)) return ORTHO_B200_ERR_SHAPE;
    for (int64_t s : {c.k_head_stride, c.v_head_stride, c.ks_head_stride, c.vs_head_stride}) if (expanded(c.kv_heads, s)) return ORTHO_B200_ERR_SHAPE;
    return ORTHO_B200_OK;
}

}  // namespace ob
