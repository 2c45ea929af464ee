// CPU check of the rows that blocks share: every row once, pieces of at most `most` rows, and nothing asked of a block without any (an
// integer division by zero ends this program).  Built and run by tests/test_row_slice.py.
#include <cstdio>
#include <initializer_list>

#include "../mixture-of-kittens_b200/csrc/row_slice.cuh"

int main() {
    for (int rows : {1, 63, 64, 128, 147, 148, 149, 192, 320, 2048, 7168, 16384})
        for (int blocks : {1, 2, 132, 148, 296})
            for (int most : {8, 16}) {
                int next = 0;
                for (int block = 0; block < blocks; ++block) {
                    const mok::RowSlice s(rows, most, block, blocks);
                    for (int early : {1, s.pieces}) {   // weights that are fetched before anything else
                        int at = s.first;
                        for (int i = 0; i < s.at_most(early); ++i) {
                            const int row = s.row(i), count = s.row(i + 1) - row;
                            if (row != at || count <= 0 || count > most || row + count > s.end) {
                                std::printf("FAILED: rows %d blocks %d block %d piece %d: [%d, %d)\n", rows, blocks, block, i, row, row + count);
                                return 1;
                            }
                            at += count;
                        }
                        if (early == s.pieces && at != s.end) return std::printf("FAILED: rows %d block %d ends at %d\n", rows, block, at), 1;
                    }
                    if (s.first != next) return std::printf("FAILED: rows %d block %d begins at %d\n", rows, block, s.first), 1;
                    next = s.end;
                }
                if (next != rows) return std::printf("FAILED: rows %d, %d are shared\n", rows, next), 1;
            }
    std::printf("ok\n");
    return 0;
}
