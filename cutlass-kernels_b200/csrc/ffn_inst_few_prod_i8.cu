#include "ffn_few_sm100.cuh"
namespace cfk {
template int allow_few_product<kProductI8>();
template int launch_few_product<kProductI8>(const ProductMaps&, const ProductParams&, const FewPlan&, cudaStream_t);
}
