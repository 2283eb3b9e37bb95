// rp_id.hip — the library's source id, in a translation unit of its own: it is the only one that
// changes when any source does.
#include "../../include/rp.h"

// The sha256 prefix of every source this library was compiled from (build.py passes it as
// RP_SRC_SHA16 and also finds it in the binary through the marker), so a benched or tested number
// names the binary that produced it and a stale build is refused (build.py / _native.load).
#ifndef RP_SRC_SHA16
#define RP_SRC_SHA16 "unknown"
#endif
__attribute__((used)) static const char kBuildMarker[] = "rp-src-sha16:" RP_SRC_SHA16;
// the compiler identity hash (build.py compiler_hash) the source id above includes: the loader
// recomputes the id with it instead of running the compiler
#ifndef RP_CC_SHA16
#define RP_CC_SHA16 "unknown"
#endif
__attribute__((used)) static const char kCcMarker[] = "rp-cc-sha16:" RP_CC_SHA16;

extern "C" const char* rp_build_id(void) { return kBuildMarker + 13; }
