// The process's choice of programmatic dependent launch.
#pragma once

#include <cstdlib>

namespace og {

// Whether a launch may begin its set-up before the stream's previous one has
// ended (every kernel here waits for that before it touches memory).
// OPENGEMM_PDL=0 turns it off for all of them, which takes launches apart when a
// fault or a profile is being looked for.
inline bool dependent_launches() {
  static const bool on = [] { const char* e = std::getenv("OPENGEMM_PDL"); return !(e && e[0] == '0'); }();
  return on;
}

}  // namespace og
