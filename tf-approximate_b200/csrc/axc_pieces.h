// Sizes that a call's workspace and its launches have to agree on: the partial sums of columns, and the pieces of the classes.  Plain
// host arithmetic, in a header of its own so that it can be checked without a GPU over any number of sizes.
#pragma once
#include <stddef.h>

namespace axc {

constexpr int kShares = 64;                    // blocks that share the rows of the output gradient's pass, at most

// Blocks that share the rows: about eight blocks for every SM, of at least 32 rows each.  Falls in steps as the columns grow, so the
// partial sums of fewer columns may take more room.
inline int column_shares(long long rows, long long columns)
{
    long long shares = (rows + 31) / 32;
    const long long across = columns / 256 + 1, most = 1184 / across + 1;
    if (shares > most) shares = most;
    if (shares > kShares) shares = kShares;
    return int(shares < 1 ? 1 : shares);
}
// Bytes of the partial sums
inline size_t slope_scratch(long long rows, long long columns) { return size_t(column_shares(rows, columns)) * size_t(columns) * 4; }

// Classes at a time where `limit` bytes hold the gradient of their logits, 16-bit values in `planes` planes: as few pieces as the limit allows, of
// equal size but for the last, at least 256 classes.  `whole`: all classes, in whole segments.
inline long long classes_of_piece(long long rows, long long whole, int planes, size_t limit)
{
    const size_t each = size_t(rows) * 2 * size_t(planes), most = limit / (each ? each : 1) / 256 * 256;
    const long long cap = most < 256 ? 256 : (long long)most < whole ? (long long)most : whole;
    const long long pieces = (whole + cap - 1) / cap;
    return ((whole + pieces - 1) / pieces + 255) / 256 * 256;
}
// The two sizes that a walk over the classes in steps of `piece` has: a whole piece's and the last one's
struct PieceSizes {
    long long n[2];
};
inline PieceSizes piece_sizes(long long classes, long long piece)
{
    return {{piece > classes ? classes : piece, classes - (classes - 1) / piece * piece}};
}
// Partial sums of the columns of any of them
inline size_t slope_scratch_of_pieces(long long rows, long long classes, long long piece)
{
    const PieceSizes s = piece_sizes(classes, piece);
    const size_t a = slope_scratch(rows, s.n[0]), b = slope_scratch(rows, s.n[1]);
    return a > b ? a : b;
}

}  // namespace axc
