#include "attention.cuh"
template int ob::launch_attention<__half>(const ob::AttentionArgs &, const ob::AttnPlan &, cudaStream_t);
