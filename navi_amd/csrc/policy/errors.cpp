// errors.cpp — the calling thread's last failure message (host code of libnavi_policy.so).
#include <cstdarg>
#include <cstdio>

#include "navi_policy.h"

namespace navi_policy {

thread_local char g_last_error[512] = "";

int set_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int set_error(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_last_error, sizeof g_last_error, fmt, ap);
    va_end(ap);
    return code;
}

}  // namespace navi_policy

extern "C" const char* navi_policy_last_error(void) { return navi_policy::g_last_error; }
