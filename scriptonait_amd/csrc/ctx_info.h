// What entry points outside sampler_api.hip use of a context.
#pragma once
#include <stdint.h>

#include <string>

struct llmhip_ctx;

namespace llmhip {

struct CtxInfo {
  int device;
  uint32_t cus;      // the device's compute units
  uint32_t* status;  // device word of the device entries' flags
};
CtxInfo ctx_info(const llmhip_ctx* ctx);

// Sets the text that llmhip_last_error returns.
void set_last_error(const std::string& what);

}  // namespace llmhip
