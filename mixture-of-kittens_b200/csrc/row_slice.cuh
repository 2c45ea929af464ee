// Rows that are cut evenly, to the row, over blocks, and a block's share in pieces.
#pragma once

#ifdef __CUDACC__
#define MOK_SLICE_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define MOK_SLICE_HOST_DEVICE inline
#endif

namespace mok {

// Rows [first, end) of block `block`, in `pieces` pieces of at most `most` rows.  With fewer rows than blocks some blocks have no piece,
// and row() no meaning.
struct RowSlice {
    int first, end, pieces;
    MOK_SLICE_HOST_DEVICE RowSlice(int rows, int most, int block, int blocks)
        : first(static_cast<int>(static_cast<long long>(rows) * block / blocks)),
          end(static_cast<int>(static_cast<long long>(rows) * (block + 1) / blocks)), pieces((end - first + most - 1) / most) {}
    // First row of piece i, or, i = pieces, the end.
    MOK_SLICE_HOST_DEVICE int row(int i) const { return first + (end - first) * i / pieces; }
    // The first n pieces, or as many as there are.
    MOK_SLICE_HOST_DEVICE int at_most(int n) const { return n < pieces ? n : pieces; }
};

}  // namespace mok
