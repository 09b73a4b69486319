#include "ffn_few_sm100.cuh"
namespace cfk {
template int allow_few_product<kGrad>();
template int launch_few_product<kGrad>(const ProductMaps&, const ProductParams&, const FewPlan&, cudaStream_t);
}
