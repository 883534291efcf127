// i8_blocks_of_piece: every value of a row is loaded once, and nothing behind the piece that its last value lies in.
#include <stdio.h>

#include <vector>

#include "../../excalibur_amd/csrc/i8_rows.h"

int main() {
    for (int k = 1; k <= 1200; ++k) {
        const int end = (k + 15) / 16 * 16;
        std::vector<int> loaded(end + 256);
        for (int piece = 0; piece < 128; piece += 16)
            for (int b = 0; b < i8_blocks_of_piece(k, piece); ++b)
                for (int e = 0; e < 16; ++e) ++loaded[b * 128 + piece + e];
        for (int i = 0; i < (int)loaded.size(); ++i)
            if (loaded[i] != (i < end)) {
                printf("%d values: byte %d loaded %d times\n", k, i, loaded[i]);
                return 1;
            }
    }
    return 0;
}
