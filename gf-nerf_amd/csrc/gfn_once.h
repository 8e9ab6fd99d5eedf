// gfn_once.h -- one-time set-up per (call site, device) that several threads may reach at once.
#pragma once

// True where the caller has to run the (idempotent) set-up of a call site on a device itself: until a thread that has run it comes back, which
// is when its set-up is known to be complete and `seen` (the call site's own static word, one bit per device ordinal) says so to all.  A
// thread therefore never goes past a call site in front of a set-up: its own, or one that had ended.
static inline bool gfn_first_call(unsigned long long& seen, int dev) {
  const unsigned long long bit = 1ull << (dev & 63);
  if (__atomic_load_n(&seen, __ATOMIC_ACQUIRE) & bit) return false;
  struct Begun {
    const void* site;
    unsigned long long devices;
  };
  constexpr int kSites = 256;  // more than a thread meets; one that meets more runs the others' set-up each time
  static thread_local Begun begun[kSites];
  for (Begun& b : begun) {
    if (!b.site) b.site = &seen;
    if (b.site != &seen) continue;
    if (b.devices & bit) {
      __atomic_fetch_or(&seen, bit, __ATOMIC_RELEASE);
      return false;
    }
    b.devices |= bit;
    return true;
  }
  return true;
}
