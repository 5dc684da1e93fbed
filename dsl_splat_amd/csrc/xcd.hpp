// Which XCD takes which block.  Blocks b, b + 8, b + 16, ... of a launch run on
// one of the eight, each with an L2 of its own.
#pragma once

#include <cstdint>

namespace gs3d {

// A launch of groups x tiles blocks in which the tiles of a group (a range of
// rows, say, against every range of columns) read the same memory: a group runs
// on one XCD, whose L2 then holds that memory once, eight groups at a time.  The
// last groups % 8 would leave XCDs idle like that, all of them but one where
// there is one group; their tiles go round the XCDs, which thus have the same
// number of blocks to within one (us, bfloat16, dealt by eights alone and so:
// dW of 8192 rows, 2048 to 2048 channels, 2 groups of 256, 484 and 160; of 500
// 000 rows, 128 to 384, 170 groups of 3, with the slope's product 543 and 463;
// one row, 512 to 4096, 1 group of 128, 8.0 and 5.1).
struct Dealt {
    uint32_t group, tile;
};
__host__ __device__ inline Dealt deal_block(uint32_t block, uint32_t groups, uint32_t tiles) {
    const uint32_t whole = groups / 8 * 8, local = block / 8;
    if (block < whole * tiles) return Dealt{local / tiles * 8 + block % 8, local % tiles};
    return Dealt{block / tiles, block % tiles};
}

}  // namespace gs3d
