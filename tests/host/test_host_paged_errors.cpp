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

struct DevBuf {
  HipBackend &be;
  void *p = nullptr;
  DevBuf(HipBackend &b, const std::vector<float> &x) : be(b) {
    auto r = be.alloc(x.size() * 4);
    CHECK(r.ok() && be.write_buffer(r.value(), x.data(), x.size() * 4).ok(), "upload");
    p = r.ok() ? r.value() : nullptr;
  }
  ~DevBuf() { (void)be.free(p); }
};

// Tensors of a step of up to `most` tokens and angles of 64 positions.
struct Step {
  static constexpr size_t most = 80, hq = 4, hkv = 2, d = 64, positions = 64;
  std::vector<float> x;
  DevBuf q, k, v, qo, o, cs;
  Tensor tq, tk, tv, tqo, to;
  static std::vector<float> values(size_t n, uint32_t seed) {
    std::vector<float> x(n);
    for (float &y : x) seed = seed * 1664525u + 1013904223u, y = (float)(seed >> 8) / 8388608.0f - 1.0f;
    return x;
  }
  Step(HipBackend &be, uint32_t seed)
      : q(be, values(most * hq * d, seed)), k(be, values(most * hkv * d, seed + 1)), v(be, values(most * hkv * d, seed + 2)),
        qo(be, std::vector<float>(most * hq * d, 0.0f)), o(be, std::vector<float>(most * hq * d, 0.0f)), cs(be, values(positions * d, 5)),
        tq{q.p, DType::F32, {most, hq, d}, true}, tk{k.p, DType::F32, {most, hkv, d}, true}, tv{v.p, DType::F32, {most, hkv, d}, true},
        tqo{qo.p, DType::F32, {most, hq, d}, true}, to{o.p, DType::F32, {most, hq, d}, true} {}
  Status write(HipPagedKvCache &c, size_t rows = positions, size_t rot = d) {
    return c.write(0, tq, tk, tv, tqo, nullptr, nullptr, 1e-6f, (const float *)cs.p, rows, rot);
  }
};

// Positions behind the table of angles: the operator would take them for padding.
static void test_positions(HipBackend &be) {
  auto made = HipPagedKvCache::create(be, config());
  if (!made.ok()) return;
  HipPagedKvCache &c = *made.value();
  Step s(be, 1);
  CHECK(c.begin_step({40, 10, 0}).ok() && s.write(c).ok() && s.write(c, 40).ok(), "40 positions of 64, and of 40");
  CHECK(!s.write(c, 39).ok() && s.write(c, 0, 0).ok(), "40 positions of 39; without rotation there are none");
  c.end_step();
  CHECK(c.begin_step({24, 0, 0}).ok() && s.write(c).ok(), "the last of 64 positions");
  c.end_step();
  CHECK(c.begin_step({0, 1, 0}).ok() && s.write(c).ok(), "an idle request's length does not count");
  c.end_step();
  CHECK(c.begin_step({1, 1, 0}).ok() && !s.write(c).ok(), "position 64 of 64");
}

// A window beyond 32 bits is one that hides nothing.
static void test_windows(HipBackend &be) {
  auto made = HipPagedKvCache::create(be, config());
  if (!made.ok()) return;
  HipPagedKvCache &c = *made.value();
  Step s(be, 2);
  const size_t n = 44 * Step::hq * Step::d;
  std::vector<float> all(n), got(n);
  CHECK(c.begin_step({40, 4, 0}).ok() && s.write(c).ok() && c.attend(0, s.tqo, s.to).ok(), "no window");
  be.read_buffer(all.data(), s.o.p, n * 4);
  for (size_t window : {(size_t)64, (size_t)INT32_MAX, (size_t)1 << 31, ((size_t)1 << 32) + 5, SIZE_MAX}) {
    CHECK(c.attend(0, s.tqo, s.to, window).ok(), "window %zu", window);
    be.read_buffer(got.data(), s.o.p, n * 4);
    CHECK(got == all, "window %zu hides something", window);
  }
}

// A step that is abandoned leaves the cache as it was: the steps around it give the same rows as in a cache
// that never saw it.
static void test_abandoned_steps(HipBackend &be) {
  auto a = HipPagedKvCache::create(be, config()), b = HipPagedKvCache::create(be, config());
  if (!a.ok() || !b.ok()) return;
  HipPagedKvCache &plain = *a.value(), &torn = *b.value();
  const std::vector<std::vector<int32_t>> steps = {{20, 3, 0}, {1, 30, 16}, {12, 1, 1}, {1, 1, 1}};
  const std::vector<std::vector<int32_t>> lost = {{5, 50, 20}, {30, 0, 1}, {1, 20, 40}, {2, 2, 2}};
  uint32_t seed = 10;
  for (size_t i = 0; i < steps.size(); ++i) {
    Step wrong(be, seed += 3), s(be, seed += 3);
    const size_t pages = torn.free_pages(), cached = torn.cached(1);
    CHECK(torn.begin_step(lost[i]).ok() && wrong.write(torn).ok(), "step to be lost");
    CHECK(i == 3 ? torn.free_pages() == pages : torn.free_pages() < pages, "its pages");  // 35, 3 and 19 tokens fit into 3, 1 and 2
    CHECK(!torn.attend(9, wrong.tqo, wrong.to).ok() && !torn.begin_step(steps[i]).ok() && torn.abandon_step().ok(), "abandon_step");
    CHECK(torn.free_pages() == pages && torn.cached(1) == cached && torn.new_tokens() == 0, "nothing is left of it");
    CHECK(torn.abandon_step().ok() && torn.free_pages() == pages, "without a step");
    std::vector<float> out[2];
    for (HipPagedKvCache *c : {&plain, &torn}) {
      CHECK(c->begin_step(steps[i]).ok() && s.write(*c).ok() && c->attend(0, s.tqo, s.to).ok(), "step %zu", i);
      std::vector<float> &o = out[c == &torn];
      o.resize(c->new_tokens() * Step::hq * Step::d);
      be.read_buffer(o.data(), s.o.p, o.size() * 4);
      c->end_step();
    }
    CHECK(out[0] == out[1] && plain.free_pages() == torn.free_pages(), "step %zu after an abandoned one", i);
    if (i == 1) CHECK(plain.release(1).ok() && torn.release(1).ok(), "release");
  }
}

int main() {
  auto r = HipBackend::create(0);
  if (!r.ok()) {
    printf("no HIP device: %s\n", r.error().c_str());
    return 77;
  }
  test_configs(*r.value());
  test_positions(*r.value());
  test_windows(*r.value());
  test_abandoned_steps(*r.value());
  if (g_fail) {
    printf("%d check(s) FAILED\n", g_fail);
    return 1;
  }
  printf("ALL PASS: refusals of the paged cache\n");
  return 0;
}
