// Which pieces of a row of 8-bit integers are loaded. Plain C++: the kernels and a check on the CPU share it.
#pragma once

// Of a row of k values, in blocks of 128 of 8 pieces of 16: how many blocks have values in the piece that begins `piece` bytes into each. What lies behind a row's last piece may be
// the end of the memory.
constexpr int i8_blocks_of_piece(int k, int piece) {
    const int blocks = k / 128 + (k % 128 != 0);
    return (blocks - 1) * 128 + piece < k ? blocks : blocks - 1;
}
