// A wait that ends: the rule by which the threads of a CTA stop waiting for one another.  Plain functions of what they poll, so that
// they can be unit-tested without a GPU.
#pragma once

#include "ptr_check.h"

namespace hfk {

enum class WaitEnd { kDone, kStopped, kRanOut };

// Polls done() until it holds, until stop() does (another thread gave up, so what is waited for may never come), or for limit_ns.
template <typename Done, typename Now, typename Stop>
HFK_HD WaitEnd bounded_wait(Done done, Now now_ns, Stop stop, uint64_t limit_ns) {
  if (done()) return WaitEnd::kDone;
  const uint64_t t0 = now_ns();
  while (!done()) {
    if (stop()) return WaitEnd::kStopped;
    if (now_ns() - t0 > limit_ns) return WaitEnd::kRanOut;
  }
  return WaitEnd::kDone;
}

// The same for work that this CTA has issued and that reads or writes its own memory: it comes to its end whatever others gave up on,
// and the CTA may not leave before, so nothing but the limit ends the wait.
template <typename Done, typename Now>
HFK_HD bool drain(Done done, Now now_ns, uint64_t limit_ns) {
  return bounded_wait(done, now_ns, [] { return false; }, limit_ns) == WaitEnd::kDone;
}

}  // namespace hfk
