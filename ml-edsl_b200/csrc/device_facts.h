// What the host asks the driver about a device and a kernel before it launches.
// No CUDA in here: the queries are the callers'.
#pragma once

namespace b200 {

// What `ask(&n)` gives (true: the query went well), or `otherwise` where it fails
// or gives nothing. `forget` takes the error of a failing query back, so that the
// next launch's check does not report it.
template <class Ask, class Forget>
int ask_or(int otherwise, Ask ask, Forget forget) {
  int n = 0;
  if (!ask(&n)) {
    forget();
    return otherwise;
  }
  return n > 0 ? n : otherwise;
}

}  // namespace b200
