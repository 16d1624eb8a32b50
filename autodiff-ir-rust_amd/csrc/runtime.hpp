// What the operators on device arrays need of a context.
#pragma once
#include <functional>

#include "../../include/adhip.h"

namespace adhip {

// Runs `f` with the context's device current; an exception becomes the context's last error and the code 2.
int context_guarded(adhip_ctx* ctx, const std::function<void()>& f);

}  // namespace adhip
