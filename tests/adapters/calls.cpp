// Calls a low-rank entry point many times without going back to Python, so
// that two threads' calls meet. Returns how many of them failed.
#include <cstdint>

extern "C" int repeat_apply(int (*apply)(void*, void*, const void*, int32_t, int64_t, const void*, int64_t, void*,
                                         int32_t, int64_t, void*),
                            void* bank, void* plan, const void* x, const void* base, void* y, void* stream,
                            int32_t times) {
  int failed = 0;
  for (int32_t i = 0; i < times; ++i) failed += apply(bank, plan, x, 0, 0, base, 0, y, 0, 0, stream) != 0;
  return failed;
}
