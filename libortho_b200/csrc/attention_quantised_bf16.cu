#include "attention_quantised.cuh"
template int ob::launch_attention_quantised<__nv_bfloat16>(const ob::QuantisedAttentionArgs &, const ob::AttnPlan &, bool, cudaStream_t);
