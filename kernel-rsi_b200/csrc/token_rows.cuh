// token_rows.cuh - rows gathered and summed by token, shared by the embedding's gradient
// (embedding.cu) and the targets' part of the vocabulary projection's gradient (linear_ce.cu).
//
// The sum of the rows of one token has to be the same on every run, so it is taken in position order:
// the positions are sorted by token first (token_sort, stable), then cut into chunks of kChunkRows
// sorted entries, each summed by one block.  A token whose run lies inside one chunk is finished there;
// a run that crosses chunks leaves one partial row per chunk, which a second kernel adds in chunk order.
#pragma once
#include "common.cuh"

namespace krsi {
namespace tokens {

constexpr int kChunkRows = 32;

inline int64_t chunks_of(int64_t n) { return (n + kChunkRows - 1) / kChunkRows; }

// The positions of tokens[0, n) sorted by token (equal tokens in position order), those outside [0, V)
// and those equal to `skip` left out:
//   start[v] .. start[v + 1]   the sorted entries of token v (start[V] = their number)
//   pos[i], tok[i]             position and token of sorted entry i
// token_bits 32 or 64.  One kernel, no workspace beyond the outputs.
cudaError_t token_sort(const void* toks, int token_bits, int64_t n, int64_t V, int64_t skip, int* start, int* pos,
                       int* tok, cudaStream_t stream);

}  // namespace tokens
}  // namespace krsi
