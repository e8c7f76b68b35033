// Pieces of the LM head that the cross-entropy (ce.hip) and the token scores (scores.hip)
// share: the products that turn one row chunk's BF16 logit gradients into gradients of the
// hidden state and of the head weight.
#pragma once

#include "launch.h"

namespace ws {

int operand_mode(const OperandDesc& d, long rows, long k, int tile_rows);

inline long round256(long b) { return (b + 255) / 256 * 256; }

// Row length of a chunk's logits and logit gradients: the vocabulary, or, when it is no
// multiple of 8, the next multiple of 64, so that the chunk's GEMMs keep 16-byte rows and the
// vector loaders (loss and gradients of 4352 x 1280 over 10883: 2265 us on the generic kernels,
// 456 padded). The padding holds zero gradients; the products read no weight row and write no
// gradient row past the vocabulary.
inline long ce_row(long vocab) { return vocab % 8 ? (vocab + 63) / 64 * 64 : vocab; }

// Operand descriptors of one row chunk [start, start + r) of the LM head.
struct CeChunk {
  const unsigned short* hidden;  // first row of the chunk
  long ld_hidden;
  long start, r;
  long ldg;  // row length of its logits / logit gradients (ce_row, or the vocabulary)
};

// Split-K factor of a chunk's dHidden GEMM.
int ce_dh_splits(long chunk, long d, long vocab);
// dW [vocab, d] += (or, with `write`, =) the chunk's G^T @ hidden.
int ce_chunk_weight_grad(const CeChunk& c, const unsigned short* gl, long vocab, long d, float* dweight,
                         long ld_dweight, bool write, const int* skip, hipStream_t s, bool round = true);
// out = r(G [r, vocab] @ W [vocab, d]), through `partials` (splits x chunk x d) when splits > 1.
int ce_chunk_dhidden(const CeChunk& c, const unsigned short* gl, const void* weight, long ld_weight,
                     const void* weight_t, long vocab, long d, int splits, long chunk, float* partials,
                     unsigned short* out, long ld_out, const int* skip, hipStream_t s);

}  // namespace ws
