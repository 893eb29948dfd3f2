// test_paged_parts.cpp -- host-side check of the places that the threads joining the parts
// of a tile of few rows read (csrc/paged.hpp, FewPart): none lies outside the part, and the
// group reads every value of its rows once.  Needs no GPU.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../llmengine_amd/csrc/paged.hpp"

using namespace mle;

#define CHECK(cond)                                                              \
  do {                                                                           \
    if (!(cond)) {                                                               \
      std::fprintf(stderr, "CHECK failed at %s:%d: %s (D %d, bits %d)\n", __FILE__, __LINE__, \
                   #cond, D, bits);                                              \
      std::abort();                                                              \
    }                                                                            \
  } while (0)

template <int D>
static void test_places() {
  using Part = FewPart<D>;
  for (int bits = 0; bits <= 3; ++bits) {
    const int quads = Part::quads(bits);
    const int groups = quads < kAttentionThreads ? kAttentionThreads / quads : 1;
    std::vector<int> seen(Part::kBytes / 16);
    for (int tid = 0; tid < kAttentionThreads; ++tid) {
      const int group = groups > 1 ? tid / quads : 0, at = tid - group * quads;
      if (group >= groups) continue;
      const uint32_t ml = Part::ml_at(at, bits);
      CHECK(ml >= Part::kMl && ml + 8 <= Part::kBytes);
      for (int i = 0; i < Part::kQuadsOfThread; ++i) {
        const uint32_t q = Part::quad_at(at, i, bits);
        CHECK(q % 16 == 0 && q + 16 <= Part::kMl);
        if (Part::has(at, i, bits)) ++seen[q / 16];
      }
    }
    for (int c = 0; c < D / 4; ++c)
      for (int r = 0; r < kFewRows; ++r)
        CHECK(seen[c * kFewRows + r] == (r < 1 << bits ? groups : 0));
  }
  std::printf("  PASS head size %d\n", D);
}

int main() {
  std::printf("test_paged_parts:\n");
  test_places<64>();
  test_places<96>();
  test_places<128>();
  test_places<256>();
  std::printf("test_paged_parts: all passed\n");
  return 0;
}
