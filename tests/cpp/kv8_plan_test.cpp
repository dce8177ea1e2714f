// The tile counts of attention's plan (kv8_index.h) for row bounds that do not ascend: sums neither wrap
// nor fall, so that the search for a tile's sequence always ends at one that has it, or there is no plan.
#include <climits>
#include <cstdio>
#include <vector>

#include "../../dsh-moss-tts_b200/csrc/kv8_index.h"

using namespace mossgpu;

static int failures = 0;
#define EXPECT(x)                                              \
    do {                                                       \
        if (!(x)) std::printf("line %d: %s\n", __LINE__, #x), ++failures; \
    } while (0)

struct Plan {
    std::vector<uint32_t> before;  // [n + 1]
    uint64_t whole = 0;            // the sum without a limit
    uint32_t wrapped = 0;          // and as 32 bits hold it
};
static Plan plan(const std::vector<int> &row_start, int rows, int group, int block_rows, uint32_t tiles) {
    Plan p;
    uint32_t sum = 0;
    for (size_t s = 0; s + 1 < row_start.size(); ++s) {
        const RowRange r = kv8_rows(row_start[s], row_start[s + 1], rows);
        p.before.push_back(sum);
        sum = kv8_add_tiles(sum, kv8_seq_tiles(tiles, r.r1 - r.r0, group, block_rows));
        const uint64_t mine = uint64_t(tiles) * uint64_t(((r.r1 - r.r0) * group + block_rows - 1) / block_rows);
        p.whole += mine;
        p.wrapped += uint32_t(mine);
    }
    p.before.push_back(sum);
    return p;
}

int main() {
    // 2048 sequences that each claim all of 65536 rows, 8192 tiles deep: 2^36 tiles where the host counts 2^26
    std::vector<int> odd;
    for (int i = 0; i <= 4096; ++i) odd.push_back(i % 2 ? 65536 : 0);
    Plan p = plan(odd, 65536, 1, 16, 8192);
    EXPECT(p.whole == uint64_t(1) << 36 && p.wrapped == 0);
    EXPECT(p.before.back() == kKv8MaxTiles);
    for (size_t s = 0; s + 1 < p.before.size(); ++s) EXPECT(p.before[s] <= p.before[s + 1]);
    // the same claims with few tiles are counted exactly
    p = plan(odd, 65536, 1, 16, 3);
    EXPECT(p.whole == p.before.back() && p.whole < kKv8MaxTiles);
    // bounds that ascend: what the host accepts stays below the limit
    std::vector<int> even;
    for (int i = 0; i <= 4096; ++i) even.push_back(i * 16);
    p = plan(even, 65536, 4, 16, 100000);
    EXPECT(p.whole == p.before.back() && p.whole < kKv8MaxTiles);
    // single counts at the ends of their ranges
    EXPECT(kv8_seq_tiles(1u << 25, 1 << 30, 1, 4) == kKv8MaxTiles);
    EXPECT(kv8_seq_tiles(1, 1 << 30, 1, 4) == 1u << 28);
    EXPECT(kv8_seq_tiles(1u << 25, 0, 7, 4) == 0);
    EXPECT(kv8_add_tiles(kKv8MaxTiles, kKv8MaxTiles) == kKv8MaxTiles);
    EXPECT(kv8_add_tiles(kKv8MaxTiles - 1, 1) == kKv8MaxTiles && kv8_add_tiles(kKv8MaxTiles - 2, 1) == kKv8MaxTiles - 1);
    if (failures == 0) std::printf("ok\n");
    return failures != 0;
}
