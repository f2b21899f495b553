// Host-only program over the addressing that the serving kernels of the HIP library
// share (csrc/serving.h), at the largest sizes that their entry points take, against
// sums and products in 128 bits. Prints one line per failure; exit status 1 if there was one.

#include "serving.h"

#include <cstdio>

namespace {

int failures = 0;

// A head's blocks of a page, up to the largest page that the checks let through, lie one
// after the other inside the page, whatever the page's number.
void blocks_lie_inside_their_page() {
    using namespace tilemix;
    alignas(16) static const std::uint8_t any[16] = {};
    for (const int d : {8, 64, 72, 128}) {
        for (const int kv_heads : {1, 2, 7}) {
            // The largest page_size of these heads, by the checks themselves.
            long long low = 1, high = 1LL << 26;
            Cache cache{};
            while (high - low > 1) {
                const long long middle = (low + high) / 2;
                const long long tokens = middle * kCacheKeys;
                const bool fits = tokens <= 0x7fffffffLL && make_cache(cache, any, 3, static_cast<int>(tokens), kv_heads, d) == hipSuccess;
                (fits ? low : high) = middle;
            }
            const int blocks = static_cast<int>(low);
            if (make_cache(cache, any, 0x7fffffff, blocks * kCacheKeys, kv_heads, d) != hipSuccess) {
                std::printf("d = %d, %d heads: no page of %d blocks\n", d, kv_heads, blocks);
                ++failures;
                continue;
            }
            const int bytes = cache_block_bytes(cache.groups);
            if (kv_heads == 1 && static_cast<long long>(blocks) * bytes <= 0x7fffffffLL) {
                std::printf("d = %d: the largest page is under 2 GiB\n", d);
                ++failures;
            }
            for (const std::int64_t page : {std::int64_t{0}, std::int64_t{1}, cache.pages - 1}) {
                for (int step = 0; step < 64; ++step) {
                    for (const int block : {step, blocks - 1 - step, static_cast<int>(0x7fffffffLL / bytes) + step - 32}) {
                        if (block < 0 || block >= blocks) continue;
                        const __int128 expected = static_cast<__int128>(page) * cache.page_bytes + static_cast<__int128>(block) * bytes;
                        const std::int64_t at = cache_block_at(page, cache.page_bytes, block, bytes);
                        if (expected != at || at < page * cache.page_bytes || at + bytes > page * cache.page_bytes + cache.head_bytes) {
                            std::printf("d = %d, %d heads: block %d of page %lld lies at %lld\n", d, kv_heads, block,
                                        static_cast<long long>(page), static_cast<long long>(at));
                            ++failures;
                        }
                    }
                }
            }
        }
    }
}

// The last key that a row sees, for rows up to a workgroup's past a sequence's end and
// lengths up to the largest.
void rows_see_up_to_their_own_key() {
    using namespace tilemix;
    const int most = 0x7fffffff;
    for (const int q_len : {1, 2, 31, 128, 129, 1 << 20, most - 128}) {
        for (const int k_len : {0, 1, 5, 128, 1 << 20, most - 64, most - 31, most - 1, most}) {
            const int context = k_len - q_len;
            for (const int from : {0, q_len - 40, q_len - 1}) {
                for (int row = from < 0 ? 0 : from; row < from + 128; ++row) {
                    const long long end = row < q_len ? row : q_len - 1LL;
                    const long long expected = static_cast<long long>(k_len) - q_len + end;
                    if (last_seen(context, row, q_len) != expected) {
                        std::printf("row %d of %d sees key %lld of %d, not %d\n", row, q_len, expected, k_len,
                                    last_seen(context, row, q_len));
                        ++failures;
                    }
                }
            }
        }
    }
}

}  // namespace

int main() {
    rows_see_up_to_their_own_key();
    blocks_lie_inside_their_page();
    if (failures == 0) std::printf("serving rules OK\n");
    return failures ? 1 : 0;
}
