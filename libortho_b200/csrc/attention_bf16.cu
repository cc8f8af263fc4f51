#include "attention.cuh"
template int ob::launch_attention<__nv_bfloat16>(const ob::AttentionArgs &, const ob::AttnPlan &, cudaStream_t);
