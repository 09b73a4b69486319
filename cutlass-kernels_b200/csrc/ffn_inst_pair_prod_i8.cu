#include "ffn_pair_sm100.cuh"
namespace cfk {
template int allow_pair_product<kProductI8>();
template int launch_pair_product<kProductI8>(const ProductMaps&, const ProductParams&, PairPlan, cudaStream_t);
}
