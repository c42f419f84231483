// What the operators of networks over sequences check in the same way.
#pragma once
#include <vector>

#include "minerva_types.h"
#include "mnv_hip.h"

namespace minerva {
namespace hip {

inline void Ok(int status, const char* what) {
  MNV_CHECK(status == MNV_OK) << what << ": " << mnv_error_string(status);
}

// The extents that say how values lie in memory: without those that are 1.
inline std::vector<int> Layout(const std::vector<int>& dims) {
  std::vector<int> r;
  for (int d : dims)
    if (d != 1) r.push_back(d);
  return r;
}
// Whether s holds values in the order of `dims`: with these extents, or flat.
inline bool LiesAs(const Scale& s, const std::vector<int>& dims) {
  const std::vector<int> have = Layout(s.ToVector());
  long long all = 1;
  for (int d : dims) all *= d;
  return have == Layout(dims) || (have.size() == 1 && have[0] == all);
}

}  // namespace hip
}  // namespace minerva
