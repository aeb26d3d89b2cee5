// Host-checkable arithmetic of the shared-prefix attention (prefix_attention.cu): which bytes its warps share.
#pragma once

namespace ernie_b200
{
// Where 16-byte chunk `chunk` of `row` lies in a tile of weights P, 128 rows of 128 BF16: two column blocks of 128
// rows of 128 bytes, chunks swizzled within a row as the tensor cores read them. A row's sixteen chunks hold its
// weights, and between two parts 64 of its FP32 results on their way out. Both go by this one function, so that a
// softmax warp, whose rows are its own, never writes where another one's weights or results lie: nothing makes the
// warps of a tile meet between one's results and another's next weights.
constexpr int kWeightRows = 128, kWeightChunks = 16;
constexpr int weight_chunk(int row, int chunk)
{
    return (chunk >> 3) * (kWeightRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// No two chunks of the tile share a byte.
constexpr bool weight_chunks_are_apart()
{
    bool taken[kWeightRows * kWeightChunks] = {};
    for (int row = 0; row < kWeightRows; ++row)
        for (int chunk = 0; chunk < kWeightChunks; ++chunk)
        {
            const int at = weight_chunk(row, chunk);
            if (at % 16 || at < 0 || at / 16 >= kWeightRows * kWeightChunks || taken[at / 16]) return false;
            taken[at / 16] = true;
        }
    return true;
}
static_assert(weight_chunks_are_apart(), "chunks of the weights' tile");

// The parts of an item that the workers `first` to `last` left behind, at places item + first and on; a list has places
// for items + workers of them. None where the two numbers cannot be workers: they come from the workspace, which holds
// anything if a worker gave up before it reached the item.
struct PartRange
{
    int first, count;
};
constexpr PartRange parts_between(int first, int last, int workers)
{
    return first < 0 || last < first || last >= workers ? PartRange{0, 0} : PartRange{first, last - first + 1};
}
} // namespace ernie_b200
