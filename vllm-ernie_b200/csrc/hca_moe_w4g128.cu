// Expert kernels of the mixture-of-experts layer for one weight format.
#include "hca_moe_experts.cuh"

template int hca::moe_experts_pass<hca::kW4G128>(const hca::MoePass&, const hca::MoeWeights&, cudaStream_t);
