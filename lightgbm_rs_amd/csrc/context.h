// context.h — what other files of the library use of a context (capi.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/lgbm_hip.h"

namespace lgbm {
int context_device(const lgbm_hip_ctx* c);
hipStream_t context_stream(const lgbm_hip_ctx* c);
// Notes the message (for a null context: where lgbm_hip_ctx_create leaves its own) and
// returns the code.
int context_error(lgbm_hip_ctx* c, int code, const std::string& message);
}  // namespace lgbm
