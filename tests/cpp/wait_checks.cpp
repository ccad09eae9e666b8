// CPU-only checks of bounded_wait.h, compiled and run by tests/test_cpp_wait.py: a clock that advances with every look at it, and
// work that is done after some of them.
#include <cstdio>

#include "bounded_wait.h"

#define CHECK(cond)                                                \
  do {                                                             \
    if (!(cond)) {                                                 \
      std::printf("FAILED %s:%d %s\n", __FILE__, __LINE__, #cond); \
      return 1;                                                    \
    }                                                              \
  } while (0)

int main() {
  using namespace hfk;
  uint64_t clock = 0;
  int polls = 0, ready = 0;
  bool gave_up = false;
  auto now = [&] { return clock += 10; };
  auto done = [&] { return polls++ >= ready; };
  auto stop = [&] { return gave_up; };
  auto reset = [&](int n, bool failed) {
    clock = 0;
    polls = 0;
    ready = n;
    gave_up = failed;
  };
  reset(0, false);
  CHECK(bounded_wait(done, now, stop, 100) == WaitEnd::kDone && polls == 1 && clock == 0);   // at once, without a look at the clock
  reset(5, false);
  CHECK(bounded_wait(done, now, stop, 100) == WaitEnd::kDone && polls == 6);
  reset(1000, false);
  CHECK(bounded_wait(done, now, stop, 100) == WaitEnd::kRanOut && clock > 100 && polls < 20);
  reset(5, true);
  CHECK(bounded_wait(done, now, stop, 100) == WaitEnd::kStopped && polls == 2);
  reset(0, true);
  CHECK(bounded_wait(done, now, stop, 100) == WaitEnd::kDone);                               // what is there is there
  // products in flight are waited for although another thread has given up, and not for ever
  reset(5, true);
  CHECK(drain(done, now, 100) && polls == 6);
  reset(1000, true);
  CHECK(!drain(done, now, 100) && clock > 100 && polls < 20);
  std::printf("wait checks ok\n");
  return 0;
}
