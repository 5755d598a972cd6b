// Device test of the host mirror's paged cache (HipPagedKvCache, argus-engine_amd/host/argus_hip_backend.hpp):
// requests that come, grow and go over several steps and two layers; every row is compared with the CPU
// oracle's attention over that request's tokens, kept contiguously by the test.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "../../argus-engine_amd/host/argus_hip_backend.hpp"

extern "C" {
void oracle_gen_data(float *dst, int64_t n, uint32_t seed);
void oracle_f32_to_f16(const float *src, uint16_t *dst, int64_t n);
int oracle_attention_gen_scalar(const float *q, const void *k, const void *v, float *out, int hq, int hkv, int d, int len,
                                int capacity, int head_major, int kv_dtype, float *scores, int64_t stride, float softcap,
                                const int32_t *kv_index);
}

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

struct DevBuf {
  HipBackend &be;
  void *p = nullptr;
  DevBuf(HipBackend &b, size_t bytes, const void *src = nullptr) : be(b) {
    auto r = be.alloc(bytes);
    CHECK(r.ok(), "alloc");
    p = r.ok() ? r.value() : nullptr;
    if (p && src) CHECK(be.write_buffer(p, src, bytes).ok(), "upload");
  }
  ~DevBuf() { (void)be.free(p); }
};

// One head: norm, rotation by half, as the operator defines it.
static void norm_rope(const float *x, const std::vector<float> &w, const float *cs, size_t d, std::vector<float> &y) {
  double sq = 0;
  for (size_t i = 0; i < d; ++i) sq += (double)x[i] * x[i];
  const double inv = 1.0 / std::sqrt(sq / d + 1e-6);
  y.resize(d);
  for (size_t i = 0; i < d / 2; ++i) {
    const double a = x[i] * inv * w[i], b = x[i + d / 2] * inv * w[i + d / 2], c = cs[i], s = cs[d / 2 + i];
    y[i] = (float)(a * c - b * s);
    y[i + d / 2] = (float)(b * c + a * s);
  }
}

static void test_steps(HipBackend &be, bool head_major) {
  const size_t hq = 8, hkv = 2, d = 64, page = 16, seqs = 3, layers = 2, positions = 128;
  HipPagedKvCache::Config cfg;
  cfg.layers = layers, cfg.heads_q = hq, cfg.heads_kv = hkv, cfg.head_dim = d, cfg.page_size = page, cfg.n_pages = 9, cfg.max_seqs = seqs;
  cfg.max_pages_per_seq = 6, cfg.max_tokens = 80, cfg.head_major = head_major;
  auto made = HipPagedKvCache::create(be, cfg);
  CHECK(made.ok(), "create: %s", made.error().c_str());
  if (!made.ok()) return;
  HipPagedKvCache &cache = *made.value();
  std::vector<float> cs(positions * d), wq(d), wk(d);
  for (size_t p = 0; p < positions; ++p)
    for (size_t i = 0; i < d / 2; ++i) {
      const double a = p * std::pow(10000.0, -2.0 * i / d);
      cs[p * d + i] = (float)std::cos(a);
      cs[p * d + d / 2 + i] = (float)std::sin(a);
    }
  for (size_t i = 0; i < d; ++i) wq[i] = 1.0f + 0.01f * i, wk[i] = 1.2f - 0.005f * i;
  DevBuf d_cs(be, cs.size() * 4, cs.data()), d_wq(be, d * 4, wq.data()), d_wk(be, d * 4, wk.data());
  const size_t most = cfg.max_tokens;
  DevBuf d_q(be, most * hq * d * 4), d_k(be, most * hkv * d * 4), d_v(be, most * hkv * d * 4), d_qo(be, most * hq * d * 4), d_out(be, most * hq * d * 4);
  Tensor tq{d_q.p, DType::F32, {most, hq, d}, true}, tk{d_k.p, DType::F32, {most, hkv, d}, true}, tv{d_v.p, DType::F32, {most, hkv, d}, true};
  Tensor tqo{d_qo.p, DType::F32, {most, hq, d}, true}, tout{d_out.p, DType::F32, {most, hq, d}, true};
  // [layer][request]: F16 rows [token][kv head][d]
  std::vector<std::vector<std::vector<uint16_t>>> ks(layers, std::vector<std::vector<uint16_t>>(seqs)), vs = ks;

  const std::vector<std::vector<int32_t>> steps = {{20, 3, 0}, {1, 1, 33}, {1, 30, 1}, {1, 1, 1}};
  uint32_t seed = 7;
  float worst = 0;
  for (size_t n = 0; n < steps.size(); ++n) {
    const auto &len = steps[n];
    Status st = cache.begin_step(len);
    CHECK(st.ok(), "begin_step %zu: %s", n, st.error().c_str());
    if (!st.ok()) return;
    const size_t t = cache.new_tokens();
    for (size_t layer = 0; layer < layers; ++layer) {
      std::vector<float> q(t * hq * d), k(t * hkv * d), v(t * hkv * d), out(t * hq * d), y;
      oracle_gen_data(q.data(), (int64_t)q.size(), seed++);
      oracle_gen_data(k.data(), (int64_t)k.size(), seed++);
      oracle_gen_data(v.data(), (int64_t)v.size(), seed++);
      be.write_buffer(d_q.p, q.data(), q.size() * 4);
      be.write_buffer(d_k.p, k.data(), k.size() * 4);
      be.write_buffer(d_v.p, v.data(), v.size() * 4);
      st = cache.write(layer, tq, tk, tv, tqo, (const float *)d_wq.p, (const float *)d_wk.p, 1e-6f, (const float *)d_cs.p, positions, d);
      CHECK(st.ok(), "write: %s", st.error().c_str());
      st = cache.attend(layer, tqo, tout);
      CHECK(st.ok(), "attend: %s", st.error().c_str());
      be.read_buffer(out.data(), d_out.p, out.size() * 4);
      size_t at = 0;
      for (size_t s = 0; s < seqs; ++s)
        for (int32_t i = 0; i < len[s]; ++i, ++at) {
          const size_t pos = cache.cached(s) + (size_t)i;
          for (size_t h = 0; h < hkv; ++h) {
            norm_rope(&k[(at * hkv + h) * d], wk, &cs[pos * d], d, y);
            std::vector<uint16_t> half(d);
            oracle_f32_to_f16(y.data(), half.data(), (int64_t)d);
            ks[layer][s].insert(ks[layer][s].end(), half.begin(), half.end());
            oracle_f32_to_f16(&v[(at * hkv + h) * d], half.data(), (int64_t)d);
            vs[layer][s].insert(vs[layer][s].end(), half.begin(), half.end());
          }
          std::vector<float> qr(hq * d), ref(hq * d);
          for (size_t h = 0; h < hq; ++h) {
            norm_rope(&q[(at * hq + h) * d], wq, &cs[pos * d], d, y);
            std::memcpy(&qr[h * d], y.data(), d * 4);
          }
          oracle_attention_gen_scalar(qr.data(), ks[layer][s].data(), vs[layer][s].data(), ref.data(), (int)hq, (int)hkv, (int)d, (int)pos + 1,
                                      (int)pos + 1, 0, 1, nullptr, 0, 0.0f, nullptr);
          for (size_t j = 0; j < hq * d; ++j) worst = std::max(worst, std::fabs(out[at * hq * d + j] - ref[j]));
        }
    }
    CHECK(cache.release(0).ok() == false, "a request of an open step is not released");
    cache.end_step();
    if (n == 1) {  // request 1 leaves; its slot and pages serve a new one
      const size_t before = cache.free_pages();
      CHECK(cache.release(1).ok() && cache.free_pages() == before + 1 && cache.cached(1) == 0, "release");
      for (size_t layer = 0; layer < layers; ++layer) ks[layer][1].clear(), vs[layer][1].clear();
    }
  }
  CHECK(worst <= 2e-3f, "rows differ from the oracle by %g", worst);
  // what does not fit is refused and changes nothing
  const size_t before = cache.free_pages();
  CHECK(!cache.begin_step({80, 0, 0}).ok() && !cache.begin_step({60, 0, 16 * 6}).ok() && !cache.begin_step({-1, 0, 0}).ok() && !cache.begin_step({1}).ok(),
        "refusals");
  CHECK(!cache.begin_step({60, 60, 40}).ok() && cache.free_pages() == before && cache.cached(0) == 23, "a refused step changes nothing");
  CHECK(cache.begin_step({0, 0, 0}).ok() && cache.new_tokens() == 0, "an empty step");
  Tensor bad = tout;
  CHECK(!cache.attend(0, tqo, bad).ok() && !cache.attend(9, tqo, bad).ok(), "attend without a step");
  printf("[paged] %s pages: %zu steps x %zu layers, worst difference from the oracle %.2e\n", head_major ? "head-major" : "token-major", steps.size(),
         layers, worst);
}

int main() {
  auto r = HipBackend::create(0);
  if (!r.ok()) {
    printf("no HIP device: %s\n", r.error().c_str());
    return 77;
  }
  test_steps(*r.value(), true);
  test_steps(*r.value(), false);
  if (g_fail) {
    printf("%d check(s) FAILED\n", g_fail);
    return 1;
  }
  printf("ALL PASS: paged cache of the host mirror verified on-device\n");
  return 0;
}
