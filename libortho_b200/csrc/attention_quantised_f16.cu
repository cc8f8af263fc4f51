#include "attention_quantised.cuh"
template int ob::launch_attention_quantised<__half>(const ob::QuantisedAttentionArgs &, const ob::AttnPlan &, bool, cudaStream_t);
