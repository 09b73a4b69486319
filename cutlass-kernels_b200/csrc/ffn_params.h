// Parameters and launchers of the feed-forward products (ffn.cu, ffn_pair_sm100.cuh).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cfk {

// What a kernel computes; `tokens` and `channels` are the rows of activations and of weights.
enum ProductMode {
  kProductI8 = 0,   // C = scaled (A B^T), 8-bit integers
  kGated16 = 1,     // h = act(x Wg^T) * (x Wu^T), 16 bits
  kGatedI8 = 2,     // the same, 8-bit integers with scales
  kGradX = 3,       // dx = dgate Wg + dup Wu: one reduction over the channels of both
  kGradW = 4        // dw_gate = dgate^T x, dw_up = dup^T x: a batch of two products, reduced over the tokens
};

struct ProductParams {
  int rows, cols;          // of the result (kGated*: of h)
  int reduce;              // length of the reduction (kGradX: of each of its two parts)
  int tiles_r, tiles_c;    // tiles of the result
  int batches;             // 2 for kGradW
  int bf16;                // operands (16-bit modes)
  int out;                 // cfk_dtype of the results
  int act, keep;           // kGated*: activation; the pre-activations are written too
  const float* row_scale;  // integer modes: of the tokens
  const float* col_scale;  // of the channels (kGatedI8: of w_gate)
  const float* col_scale2; // kGatedI8: of w_up
  const float* bias;       // kProductI8, or null
  // A TMA store writes whole 16-byte pieces: behind the last element of a row it would put zeros up to the next multiple of 16 bytes.
  // So the descriptors of the results end at the last whole piece, column `whole`, and the columns from there on are
  // stored one by one.
  int whole;
  void* d[3];
  int64_t d_stride[3];
  int* status;
};

// Operands and results of a product.  x: tokens (kGradX: dgate, dup; kGradW: dgate, dup); y: weights (kGated*, kGradX: w_gate,
// w_up; kGradW: x); d: the result (kGated*: h, gate, up; kGradW: dw_gate, dw_up).
struct ProductMaps { CUtensorMap x[2], y[2], d[3]; };

template <int MODE>
int launch_pair_product(const ProductMaps& maps, const ProductParams& p, cudaStream_t stream);

}  // namespace cfk
