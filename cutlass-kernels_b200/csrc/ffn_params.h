// Parameters, cuts and launchers of the feed-forward products (ffn.cu, ffn_pair_sm100.cuh, ffn_few_sm100.cuh).
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
  kGrad = 3         // dx = dgate Wg + dup Wu, one reduction over the channels of both; dw_gate = dgate^T x, dw_up = dup^T x, a batch
                    // of two products reduced over the tokens
};

// Operands.  kProductI8, kGated*: x[0] tokens, y weights (w_gate, w_up).  kGrad: x dgate and dup, y w_gate, w_up and the tokens.
struct ProductMaps { CUtensorMap x[2], y[3]; };

struct ProductParams {
  int rows, cols;          // of the result (kGrad: of dx)
  int reduce;              // length of the reduction (kGrad: of each of the two parts of dx)
  int bf16;                // operands (16-bit modes)
  int out;                 // cfk_dtype of the results
  int act, keep;           // kGated*: activation; the pre-activations are written too
  const float* row_scale;  // integer modes: of the tokens
  const float* col_scale;  // of the channels (kGatedI8: of w_gate)
  const float* col_scale2; // kGatedI8: of w_up
  const float* bias;       // kProductI8, or null
  void* d[3];              // results (kGated*: h, gate, up; kGrad: dx, dw_gate, dw_up) and the distance of their rows
  int64_t d_stride[3];
  int wide;                // all rows of the results that exist start at multiples of 32 bytes
  int* status;
  unsigned long long acc_limit;      // of the wait for an accumulator, ns
};
// An accumulator takes as long as its reduction: 1 us per k-block on top of the limit of other waits, where a k-block takes 0.15 to
// 0.4 us.  A tile of 900 million tokens' weight gradients takes 3 s.
constexpr unsigned long long kNsPerBlock = 1000;

// Division of 0 <= n < 2^31 by a constant of the launch: a product and a shift (T. Granlund, P. Montgomery, Division by invariant
// integers using multiplication, 1994).
struct Divisor {
  uint32_t m, shift;
};
inline Divisor make_divisor(uint32_t d) {
  uint32_t l = 0;
  while (l < 31 && (1u << l) < d) ++l;
  return Divisor{(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1), l};
}

// One list of output tiles of the kernel on CTA pairs (256 rows x 2 bn accumulator columns each).
struct PairJob {
  int kind;                // kGrad: 0 dx, 1 dw_gate and dw_up
  int rows, cols;          // of the result
  int reduce;              // of a part of the reduction
  int bn;                  // accumulator columns per CTA: 64, 96 or 128.  A tile has bn columns of h, 2 bn of any other result
  int tiles_r, tiles_c, batches;
  Divisor per_batch, per_band, tail_rows;      // tiles of a batch, of a band of kGemmBand tile rows; tile rows of the last, shorter band
};
// The pairs take the tiles of the first list in turn.  Those that get one more of them than the others take `share` tiles of the second
// list each, the others what is left.
struct PairPlan {
  PairJob job[2];
  int jobs, pairs, share;
  int most, more;          // tiles of the first list that every pair has; pairs that have one more
  int stages, y_bytes;     // of the ring; of a k-block of Y in a stage
  int staged;              // kGrad: results pass through shared memory
};

// allow_*: the kernel's shared memory on the current device, ahead of its launch.
template <int MODE>
int allow_pair_product();
template <int MODE>
int launch_pair_product(const ProductMaps& maps, const ProductParams& p, PairPlan plan, cudaStream_t stream);

// How the kernel for few tokens cuts a product (kGrad: dx).
struct FewPlan {
  int tt;                  // tokens per tile; 0: the product runs on CTA pairs
  int splits;              // CTAs of a cluster that share a tile's reduction, 1..8
  int stages;              // of the ring
  int tiles_ch, tiles_tok; // tiles of 128 channels x tt tokens
};
constexpr int kFewMaxStages = 12, kFewHead = 1024 + 256;                     // alignment slack and the barrier block
constexpr int kFewSmemHalf = 113 * 1024, kFewSmemFull = 226 * 1024;          // bytes of a CTA: two per SM, one per SM
constexpr int few_weights(int mode) { return mode == kGated16 || mode == kGatedI8 ? 2 : 1; }   // weights a tile reads per k-block

template <int MODE>
int allow_few_product();
template <int MODE>
int launch_few_product(const ProductMaps& maps, const ProductParams& p, const FewPlan& f, cudaStream_t stream);

}  // namespace cfk
