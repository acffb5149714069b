// Check of the C++ face of the calls on a 4- or 8-bit cache
// (include/kvbridge/attention_ext.h): sizes and the exception types of what is
// refused.  No device call: every launch below is rejected on the host before
// anything is enqueued.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <stdexcept>
#include <string>

#include "kvbridge/attention_ext.h"

static int failures = 0;
static void expect(bool ok, const char* what) {
  if (!ok) {
    std::fprintf(stderr, "FAIL: %s\n", what);
    ++failures;
  }
}

template <class F>
static std::string invalid_message(F&& f) {
  try {
    f();
  } catch (const std::invalid_argument& e) {
    return e.what();
  } catch (...) {
    return "<other exception>";
  }
  return "<no exception>";
}

int main() {
  using namespace kvbridge;
  void* fake = reinterpret_cast<void*>(0x1000);
  float* f = static_cast<float*>(fake);
  uint32_t* u = static_cast<uint32_t*>(fake);
  const int64_t* i64 = static_cast<const int64_t*>(fake);

  const AppendShape as{4, 8, 128, 64, 10, 1024, 1024, SourceType::f16};
  expect(append_i4_error(as) == nullptr, "valid append shape");
  AppendShape as_bad = as;
  as_bad.dim = 96;
  expect(std::string(append_i4_error(as_bad)) == "dim must be 64, 128 or 256", "append dim");
  expect(invalid_message([&] { append_kv_i4(as, fake, fake, nullptr, nullptr, nullptr, u, u, nullptr); }) ==
             "append buffers must be non-null",
         "append null slots");

  const ReadShape rs{4, 8, 128, 64, 10, 4, OutputType::bf16};
  expect(read_shape_error(rs) == nullptr, "valid read shape");
  expect(invalid_message([&] { read_kv(rs, u, nullptr, fake, fake, fake, fake, fake, nullptr); }) ==
             "cache buffers must be non-null",
         "read null pool");

  const ScoredShape ss{4, 5, 32, 8, 128, 64, 8192, 131072, 4 * 131072, 8192, 2048, 4, SourceType::bf16, 32 * 128, 0, 0.088f, 0.f};
  expect(scored_shape_error(ss) == nullptr, "valid scored shape");
  expect(scored_item_count(ss) == 4 * 64, "items");
  expect(scored_scratch_elements(ss) == size_t(4) * 64 * 5 * 32 * 130, "scratch elements");
  expect(scored_counter_elements(ss) == 4 * 8 * 2, "counter elements");
  ScoredShape ss_bad = ss;
  ss_bad.cap = -1.f;
  expect(invalid_message([&] { (void)scored_item_count(ss_bad); }) == "score cap must be finite and not negative", "cap");
  const ScoredInput in{fake, i64, u, u, i64, u, fake, fake, fake, fake, nullptr, nullptr};
  expect(invalid_message([&] { decode_attention_scored(ss, in, f, nullptr, f, f, fake, OutputType::none, nullptr); }) ==
             "unknown output type",
         "output type");
  expect(invalid_message([&] { accumulate_weights(ss, in, f, f, 1, nullptr, nullptr); }) ==
             "m, l and weights must be non-null device buffers",
         "weights buffer");

  const EvictShape es{2, 8, 128, 16, 500, 4000, 8000, 500, 100, 100, 4, 20, 4};
  expect(evict_shape_error(es) == nullptr, "valid evict shape");
  expect(evict_scratch_elements(es) >= 2 * 4000, "evict scratch");
  const EvictInput ei{u, u, u, nullptr};
  expect(invalid_message([&] { evict_select(es, ei, nullptr, u, u, u, nullptr); }) == "eviction buffers must be non-null",
         "select buffers");
  const EvictCache ec{fake, fake, fake, fake, nullptr, u, u, static_cast<int64_t*>(fake)};
  expect(invalid_message([&] { evict_move(es, ei, ec, u, u, nullptr); }) == "positions need k_positions", "move positions");
  if (failures) return 1;
  std::printf("PASS C++ API of the 4- and 8-bit cache\n");
  return 0;
}
