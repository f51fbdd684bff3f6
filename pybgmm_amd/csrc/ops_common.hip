// Error reporting of libbgmm_ops.so and the runtime it is bound to.
#include "ops_common.h"

#include <cstdarg>
#include <cstdio>
#include <dlfcn.h>

static thread_local char g_ops_error[512];

int ops_fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_ops_error, sizeof g_ops_error, fmt, ap);
    va_end(ap);
    return code;
}

int ops_launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return BGMM_OPS_OK;
    return ops_fail(BGMM_OPS_EDEVICE, "%s: %s", what, hipGetErrorString(e));
}

extern "C" const char *bgmm_ops_last_error(void) { return g_ops_error; }

extern "C" const char *bgmm_ops_runtime_path(void) {
    Dl_info info;
    return dladdr((void *)&hipGetDeviceCount, &info) && info.dli_fname ? info.dli_fname : "";
}
