// Device test of the host mirror's paged cache (HipPagedKvCache) where a call cannot be served: what it refuses,
// and what it leaves behind.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "../../argus-engine_amd/host/argus_hip_backend.hpp"

using namespace argus;

static int g_fail = 0;
#define CHECK(cond, ...)                                       \
  do {                                                         \
    if (!(cond)) {                                             \
      printf("FAIL %s:%d: ", __FILE__, __LINE__);              \
      printf(__VA_ARGS__);                                     \
      printf("\n");                                            \
      ++g_fail;                                                \
    }                                                          \
  } while (0)

static HipPagedKvCache::Config config() {
  HipPagedKvCache::Config c;
  c.layers = 1, c.heads_q = 4, c.heads_kv = 2, c.head_dim = 64, c.page_size = 16, c.n_pages = 12, c.max_seqs = 3;
  c.max_pages_per_seq = 6, c.max_tokens = 80;
  return c;
}

// A cache whose sizes no step could use is not made.
static void test_configs(HipBackend &be) {
  CHECK(HipPagedKvCache::create(be, config()).ok(), "the plain configuration");
  for (size_t page : {0u, 8u, 24u, 2048u}) {
    HipPagedKvCache::Config c = config();
    c.page_size = page;
    CHECK(!HipPagedKvCache::create(be, c).ok(), "page_size %zu", page);
  }
  for (size_t d : {0u, 32u, 96u, 512u}) {
    HipPagedKvCache::Config c = config();
    c.head_dim = d;
    CHECK(!HipPagedKvCache::create(be, c).ok(), "head_dim %zu", d);
  }
  HipPagedKvCache::Config c = config();
  c.heads_q = 5;
  CHECK(!HipPagedKvCache::create(be, c).ok(), "5 heads over 2");
}

int main() {
  auto r = HipBackend::create(0);
  if (!r.ok()) {
    printf("no HIP device: %s\n", r.error().c_str());
    return 77;
  }
  test_configs(*r.value());
  if (g_fail) {
    printf("%d check(s) FAILED\n", g_fail);
    return 1;
  }
  printf("ALL PASS: refusals of the paged cache\n");
  return 0;
}
