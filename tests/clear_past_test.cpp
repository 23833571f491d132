// Rows of a tile of V past a sequence's end (csrc/paged_kernel.h: paged_clear_past), on the host: what a wave goes by while another one is
// clearing them; run by tests/test_clear_past.py.
#include "paged_kernel.h"

#include <cstdio>
#include <vector>

// A wave's stores land in their order, one KiB each.  Whatever of another wave's has landed when a wave looks, it has to see what is left to clear.
template <int D>
static int seen_in_time()
{
    using T = fa::PagedTile<D>;
    constexpr int per = 1024 / T::ROW;  // rows of a store
    for (int left = 1; left < T::BC; ++left) {
        const int stores = (T::BC - left + per - 1) / per;
        for (int landed = 0; landed < stores; ++landed) {
            std::vector<bool> odd(T::BC, false);  // rows that are not finite: the last key's and those that repeat it
            for (int r = left - 1; r < T::BC; ++r) odd[r] = r < left || r >= left + landed * per;
            const int asked = fa::paged_asked_row(left);
            if (asked < 0 || asked >= T::BC || !odd[asked]) {
                std::printf("D %d: %d keys of the tile, %d of %d stores landed: row %d does not tell\n", D, left, landed, stores, asked);
                return 1;
            }
        }
    }
    return 0;
}

int main() { return seen_in_time<64>() || seen_in_time<128>(); }
