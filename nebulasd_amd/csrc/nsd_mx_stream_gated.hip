// The stream kernel's gated forms (nsd_mx_stream.h).
#include "nsd_mx_stream.h"

namespace nsd {

int mx_stream_gated(const MxArgs& a, const MxConfig& c, hipStream_t st) {
  return launch_mx_rows<true>(std::make_integer_sequence<int, 8>{}, a, c, st);
}

}  // namespace nsd
