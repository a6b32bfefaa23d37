// What the translation units of the C ABI share.
#ifndef JPP_API_H
#define JPP_API_H

namespace jpp_api {

// leaves the message for jppgpu_last_error on this thread, returns `code`
int fail(int code, const char* msg) noexcept;

}  // namespace jpp_api

#endif  // JPP_API_H
