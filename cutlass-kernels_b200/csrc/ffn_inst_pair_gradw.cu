#include "ffn_pair_sm100.cuh"
namespace cfk {
template int launch_pair_product<kGradW>(const ProductMaps&, const ProductParams&, cudaStream_t);
}
