// paged_records.h -- where the query rows of a cut query tile lie in its partial records
// (paged_attn.cu): host and device arithmetic in one place, with no other header, so that it can
// be enumerated on the CPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define MLZC_REC __host__ __device__ __forceinline__
#else
#define MLZC_REC inline
#endif

namespace mlzc {
namespace paged {

// A record holds the rows of a piece without gaps, tokens outermost: (token in the piece) * G +
// (head in the group).  A query tile fills tq * G of the 128 rows of the products, fewer where G
// does not divide 128, so its rows' places follow on the tile's before.
//
// Rows of a record: of a call with `tokens` new tokens in all, G query heads a KV head, query
// tiles of tq tokens, ns of them a piece.
MLZC_REC int record_rows(int64_t tokens, int G, int tq, int ns) {
    const int64_t most = (int64_t)tq * ns;
    return (int)(tokens < most ? tokens : most) * G;
}
// The place of row `row` of the piece's query tile `tile`.
MLZC_REC int record_row(int tile, int row, int tq, int G) { return tile * tq * G + row; }

}  // namespace paged
}  // namespace mlzc
