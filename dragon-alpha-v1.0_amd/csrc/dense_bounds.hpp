// Where the buffer descriptors of the bf16 tile kernel end: plain arithmetic, no device code, so that it can be tried on the host.
#pragma once

namespace alpha {

// Bytes from a tile's first element of a step to the operand's end, for rows `ld` elements apart that are whole 16-byte chunks
// long; `krem` k are left from the step's first on (<= 0: none, and nothing may be read). A lane reads 16 bytes at row * ld * 2 + ..,
// and one whose row or k the operand does not have must come to lie behind the end: there the hardware gives zeros.

// k along the rows, `rows` >= 1 of them in the tile, 32 k a step. The end is that of the last row's chunks, not 32 k behind
// its beginning: with rows 8, 16 or 24 apart the next rows' places would lie before that, behind the operand.
constexpr unsigned tile_end_straight(int rows, unsigned ld, int krem)
{
    const int k = krem < 32 ? (krem > 0 ? (krem + 7) & ~7 : 0) : 32;
    return ((unsigned)(rows - 1) * ld + (unsigned)k) * 2;
}
// k as the rows, 32 of them a step, `columns` from the tile's first on.
constexpr unsigned tile_end_t(int columns, unsigned ld, int krem)
{
    return krem > 0 ? ((unsigned)((krem < 32 ? krem : 32) - 1) * ld + (unsigned)((columns + 7) & ~7)) * 2 : 0u;
}

}  // namespace alpha
