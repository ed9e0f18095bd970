// Host run of the 8-bit cache's index and scale arithmetic (csrc/kv8.h) over a sweep of sizes:
// scales against a search, page slots against a token-by-token walk, the split of the line of
// tiles, shared-memory offsets and the permutation of score columns.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <set>
#include <vector>

#include "../../tiledattention_b200/csrc/kv8.h"

using namespace ta::kv8;

static int checks = 0;
#define CHECK(c)                                            \
  do {                                                      \
    ++checks;                                               \
    if (!(c)) {                                             \
      std::printf("FAIL line %d: %s\n", __LINE__, #c);      \
      return 1;                                             \
    }                                                       \
  } while (0)

static uint32_t bits(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  return u;
}

template <int COLS, int PLANE>
static bool offsets_fit(int rows, int chunks) {
  std::set<uint32_t> seen;
  for (int r = 0; r < rows; ++r)
    for (int c = 0; c < chunks; ++c) {
      const uint32_t at = chunk_at<COLS, PLANE>(r, c);
      if (at % 16 || at + 16 > static_cast<uint32_t>(rows * chunks * 16) || !seen.insert(at).second)
        return false;
      ++checks;
    }
  for (int c = 0; c < chunks; ++c)  // 8 rows of one ldmatrix phase, in and out of order
    for (int r0 = 0; r0 < rows; r0 += 16)
      for (int half = 0; half < 2; ++half) {
        std::set<uint32_t> banks, keys;
        for (int r = 0; r < 8; ++r) {
          banks.insert(chunk_at<COLS, PLANE>(r0 + key_at(8 * half + r), c) % 128);
          keys.insert(chunk_at<COLS, PLANE>(r0 + key_of_column(r, half), c) % 128);
        }
        if (banks.size() != 8 || keys.size() != 8) return false;
      }
  return true;
}

int main() {
  // scales: the least power of two that holds amax, at and around every border
  for (int e = -140; e <= 127; ++e)
    for (float f : {1.0f, 1.5f, 1.7499999f, 1.75f, 1.7500001f, 1.99f}) {
      const float a = std::ldexp(f, e);
      if (!std::isfinite(a)) continue;
      int want = kScaleExpMin;
      while (want < kScaleExpMax && std::ldexp(448.0, want) < static_cast<double>(a)) ++want;
      CHECK(scale_exponent(bits(a)) == want);
    }
  CHECK(scale_exponent(0) == kScaleExpMin);
  for (int e = kScaleExpMin; e <= kScaleExpMax; ++e) CHECK(stored_exponent(bits(std::ldexp(1.f, e))) == e);
  CHECK(stored_exponent(0) == kScaleExpMin && stored_exponent(0x7fffffffu) == kScaleExpMax &&
        stored_exponent(0xffffffffu) == kScaleExpMax);

  // page ids
  const int32_t row[4] = {3, -1, 7, 2147483647};
  CHECK(checked_page(row, 0, 4, 8) == 3 && checked_page(row, 2, 4, 8) == 7);
  CHECK(checked_page(row, 1, 4, 8) == -1 && checked_page(row, 3, 4, 8) == -1);
  CHECK(checked_page(row, 2, 4, 7) == -1);
  CHECK(checked_page(row, 4, 4, 8) == -1 && checked_page(row, -1, 4, 8) == -1);

  // slots: every token of a write in exactly one row, rows in bounds
  for (int page : {16, 32, 64, 128})
    for (int start : {0, 1, 15, 16, 17, 63, 64, 127, 128, 1000})
      for (int count : {0, 1, 2, 15, 16, 17, 130, 333}) {
        const int slots = (count + page - 2) / page + 1;
        int next = 0;
        for (int s = 0; s < slots; ++s) {
          const int64_t slot = start / page + s;
          const SlotSpan sp = slot_span(start, count, slot, page);
          if (sp.row1 <= sp.row0) continue;
          CHECK(sp.row0 >= 0 && sp.row1 <= page && sp.t0 == next);
          CHECK(slot * page + sp.row0 == start + next);
          CHECK(s == 0 || sp.row0 == 0);
          next += sp.row1 - sp.row0;
        }
        CHECK(next == count);
      }

  // extents and row limits stay in range
  for (int length : {-5, 0, 1, 100, 2147483647})
    for (int count : {-3, 0, 1, 5, 9}) {
      const SeqExtent e = checked_extent(length, count, 5, 128);
      CHECK(e.length >= 0 && e.length <= 128 && e.count >= 0 && e.count <= 5);
      CHECK(e.bad == (length < 0 || length > 128 || count < 0 || count > 5));
      for (int t = 0; t < 5; ++t)
        for (int causal : {0, 1}) {
          const int lim = row_limit(e.length, e.count, t, causal);
          CHECK(lim >= 0 && lim <= e.length);
          if (t < e.count && t == e.count - 1) CHECK(lim == e.length);
          if (t >= e.count) CHECK(lim == 0);
        }
    }

  // division by the group: every group, at its multiples' borders up to 2^24
  for (int g = 1; g <= kMaxGroup; ++g)
    for (int n = 0; n < (1 << 24); n += n < 4096 ? 1 : 65521)
      for (int m : {n, n / g * g, n / g * g + g - 1})
        if (m < (1 << 24) && divide_by_group(m, group_reciprocal(g)) != m / g) CHECK(false);
  CHECK(divide_by_group((1 << 24) - 1, group_reciprocal(256)) == ((1 << 24) - 1) / 256);

  // tiles of a block of rows: the last key that any of its rows sees, against a walk over rows
  for (int group : {1, 3, 4, 8})
    for (int T : {1, 5, 64, 100})
      for (int length : {0, 1, 60, 129, 1000})
        for (int count : {0, 1, 3, 100})
          for (int causal : {0, 1})
            for (int n : {128, 256}) {
              if (count > T) continue;
              const SeqExtent e = checked_extent(length, count, T, 1 << 20);
              for (int row0 = 0; row0 < group * T + n; row0 += n) {
                int lim = 0;
                for (int r = row0; r < row0 + n && r < group * T; ++r) {
                  const int l = row_limit(e.length, e.count, r / group, causal);
                  if (l > lim) lim = l;
                }
                CHECK(block_tiles(e, group * T, group_reciprocal(group), row0, n, causal, 128) == (lim + 127) / 128);
              }
            }

  // runs: they tile the line, none empty, and run_of finds the run of every tile
  for (int64_t total : {1, 2, 7, 295, 296, 297, 1000, 4096, 100003})
    for (int64_t grid : {1, 3, 148, 296}) {
      const int64_t parts = grid < total ? grid : total;
      int64_t i = 0;
      for (int64_t w = 0; w < total; ++w) {
        while (run_begin(i + 1, total, parts) <= w) ++i;
        if (run_of(w, total, parts) != i || run_begin(i, total, parts) > w) CHECK(false);
      }
      CHECK(run_begin(0, total, parts) == 0 && run_begin(parts, total, parts) == total);
      for (int64_t r = 0; r < parts; ++r)
        CHECK(run_begin(r, total, parts) < run_begin(r + 1, total, parts));
    }

  CHECK((offsets_fit<64, 0>(32, 4)));
  CHECK((offsets_fit<64, 0>(16, 4)));
  CHECK((offsets_fit<128, 0>(32, 8)));
  CHECK((offsets_fit<128, 0>(16, 8)));
  CHECK((offsets_fit<128, 16 * 128>(16, 16)));

  // score columns: each key of 16 once, columns 2t, 2t+1 of the halves at positions 4t .. 4t+3
  std::set<int> keys;
  for (int half = 0; half < 2; ++half)
    for (int n = 0; n < 8; ++n) keys.insert(key_of_column(n, half));
  CHECK(keys.size() == 16 && *keys.begin() == 0 && *keys.rbegin() == 15);
  for (int t = 0; t < 4; ++t)
    for (int half = 0; half < 2; ++half) {
      CHECK(key_of_column(2 * t, half) == key_at(4 * t + 2 * half));
      CHECK(key_of_column(2 * t + 1, half) == key_of_column(2 * t, half) + 1);
    }
  std::printf("ok %d\n", checks);
  return 0;
}
