// Which bytes of the weights' tile each softmax warp of the shared-prefix attention touches (no GPU): a warp stores its
// 32 rows' weights, and between two parts its rows' results, and no barrier stands between one warp's results and
// another's next weights, so the warps' bytes may not meet. And where the join looks for an item's parts, whatever the
// workspace holds in their workers' place.
#include "attend_layout.h"
#include <climits>
#include <cstdio>
#include <vector>

using namespace ernie_b200;

namespace
{
constexpr int kTileBytes = kWeightRows * kWeightChunks * 16;

// The bytes of one warp's rows, chunk by chunk, by any placement of its results.
template <class Place> std::vector<char> bytes_of(int warp, Place place)
{
    std::vector<char> taken(kTileBytes, 0);
    for (int row = 0; row < 32; ++row)
        for (int chunk = 0; chunk < kWeightChunks; ++chunk)
        {
            const int at = place(warp, row, chunk);
            for (int i = 0; i < 16; ++i) taken.at(at + i) = 1;
        }
    return taken;
}

int own_rows(int warp, int row, int chunk) { return weight_chunk(warp * 32 + row, chunk); }
// A placement that this check has to find fault with: each warp's results in a quarter of the tile's bytes.
int by_quarters(int warp, int row, int chunk) { return warp * 8192 + row * 256 + ((chunk ^ (row & 15)) << 4); }

template <class Place> int clashes(Place results)
{
    int found = 0;
    for (int warp = 0; warp < 4; ++warp)
    {
        const auto mine = bytes_of(warp, results);
        for (int other = 0; other < 4; ++other)
        {
            if (other == warp) continue;
            const auto weights = bytes_of(other, own_rows), staged = bytes_of(other, results);
            for (int i = 0; i < kTileBytes; ++i) found += mine[i] && (weights[i] || staged[i]);
        }
    }
    return found;
}

// The join reads places item + first .. + count - 1 of items + workers.
bool parts_stay_inside()
{
    const int anything[] = {INT_MIN, INT_MIN + 1, -1, 0, 1, 2, 7, 8, 9, 147, 148, 149, 1183, 1184, 1185, 0x3f800000, 0x7f7fffff, INT_MAX - 1, INT_MAX};
    for (int workers : {1, 2, 8, 148, 1184})
        for (int first : anything)
            for (int last : anything)
            {
                const PartRange r = parts_between(first, last, workers);
                const bool real = 0 <= first && first <= last && last < workers;
                if (r.count < 0 || r.first < 0 || r.first > workers - r.count) return false;
                if (real ? r.first != first || r.count != last - first + 1 : r.count != 0) return false;
            }
    return true;
}
} // namespace

int main()
{
    if (!parts_stay_inside()) return std::fprintf(stderr, "an item's parts lie outside the list\n"), 1;
    const auto all = [] {
        std::vector<char> sum(kTileBytes, 0);
        for (int warp = 0; warp < 4; ++warp)
        {
            const auto one = bytes_of(warp, own_rows);
            for (int i = 0; i < kTileBytes; ++i) sum[i] += one[i];
        }
        return sum;
    }();
    for (char times : all)
        if (times != 1) return std::fprintf(stderr, "a byte of the tile belongs to %d warps\n", times), 1;
    if (clashes(own_rows) != 0) return std::fprintf(stderr, "a warp's results lie on another's bytes\n"), 1;
    if (clashes(by_quarters) == 0) return std::fprintf(stderr, "the check sees no clash where there is one\n"), 1;
    std::puts("attention layout passed");
    return 0;
}
