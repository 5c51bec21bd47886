// tile_rows.h -- which rows a tile reads where it reaches past its interval.
// Plain arithmetic, for the kernels and for checks on a host.
#ifndef TRW_TILE_ROWS_H
#define TRW_TILE_ROWS_H

namespace trw {
namespace ops {

// Rows first .. first + rows - 1 of a tile as bytes from row `from`, its nearest
// row inside [begin, end): each row kept between `from` and the last one.
struct EdgeRows {
    int before;  // bytes from row `first` to row `from`
    int last;    // bytes from row `from` to the last row that a tile can name
};
// rows * pitch fits 31 bits (checked on the host); a whole interval need not:
// where the tile starts before it, `last` is one of the tile's rows all the same.
constexpr EdgeRows edge_rows(int first, int from, int end, int rows, int pitch) {
    return EdgeRows{(from - first) * pitch,
                    (end - 1 - from < rows - 1 ? end - 1 - from : rows - 1) * pitch};
}
// `row`: bytes from row `first` to the tile's row.
constexpr int edge_row(const EdgeRows& e, int row) {
    return row - e.before < 0 ? 0 : row - e.before > e.last ? e.last : row - e.before;
}

}  // namespace ops
}  // namespace trw
#endif  // TRW_TILE_ROWS_H
