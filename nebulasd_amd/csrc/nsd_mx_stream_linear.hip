// The stream kernel's plain forms (nsd_mx_stream.h).
#include "nsd_mx_stream.h"

namespace nsd {

int mx_stream_linear(const MxArgs& a, const MxConfig& c, hipStream_t st) {
  return launch_mx_rows<false>(std::make_integer_sequence<int, 8>{}, a, c, st);
}

}  // namespace nsd
