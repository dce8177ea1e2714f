// The index checks of the 8-bit cache (kv8_index.h): whatever device memory holds, a row range
// stays inside the rows, a position inside its slot, a page inside the pool, and the last byte of
// the last cell inside codes and scales.
#include <climits>
#include <cstdio>
#include <initializer_list>

#include "../../dsh-moss-tts_b200/csrc/kv8_index.h"

using namespace mossgpu;

static int failures = 0;
#define EXPECT(x)                                              \
    do {                                                       \
        if (!(x)) std::printf("line %d: %s\n", __LINE__, #x), ++failures; \
    } while (0)

int main() {
    const int odd[] = {INT_MIN, -100, -1, 0, 1, 3, 15, 16, 17, 63, 64, 65, 100, INT_MAX - 16, INT_MAX};
    for (int a : odd)
        for (int b : odd)
            for (int rows : {1, 4, 1000}) {
                const RowRange r = kv8_rows(a, b, rows);
                EXPECT(r.r0 >= 0 && r.r0 <= r.r1 && r.r1 <= rows);
                if (a >= 0 && a <= b && b <= rows) EXPECT(r.r0 == a && r.r1 == b);
            }
    mossgpu_kv8_cache c{};
    c.n_pages = 7, c.n_slots = 3, c.pages_per_slot = 4, c.kv_heads = 5, c.head_dim = 64;
    for (int slot : odd)
        for (int ctx : odd)
            for (int n : {0, 1, 16, 64, 65, INT_MAX}) {
                int status = 0;
                const SeqSpan s = kv8_span(c, slot, ctx, n, &status);
                const int cap = slot >= 0 && slot < 3 ? 64 : 0;
                EXPECT(s.ctx >= 0 && s.ctx <= s.total && s.total <= cap);
                const bool fits = cap > 0 && ctx >= 0 && ctx <= cap && n <= cap - ctx;
                if (fits) EXPECT(s.ctx == ctx && s.total == ctx + n && status == 0);
                if (!fits && (cap > 0 || n > 0)) EXPECT(status == kStatusBadPosition);
            }
    for (int page : odd) {
        int status = 0;
        const int got = kv8_page(c, page, &status);
        EXPECT(page >= 0 && page < 7 ? got == page && status == 0 : got == -1 && status == kStatusBadPage);
    }
    EXPECT(kv8_cell(c, 0, 0, 0, 0) == 0);
    EXPECT(kv8_cell(c, 6, 1, 4, 15) == size_t(7) * 2 * 5 * 16 - 1);
    size_t next = 0;  // cells are numbered without gaps in the order of the layout
    for (int p = 0; p < 7; ++p)
        for (int h = 0; h < 2; ++h)
            for (int k = 0; k < 5; ++k)
                for (int o = 0; o < 16; ++o) EXPECT(kv8_cell(c, p, h, k, o) == next++);
    c.n_pages = INT_MAX, c.kv_heads = 4096;  // far past 32 bits
    EXPECT(kv8_cell(c, INT_MAX - 1, 1, 4095, 15) == size_t(INT_MAX) * 2 * 4096 * 16 - 1);
    if (failures == 0) std::printf("ok\n");
    return failures != 0;
}
