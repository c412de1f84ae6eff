/*
 * r9vx_host.h -- what the C-ABI sources share: collecting every problem of a
 * call before it is refused, and the text of the last error.
 */
#ifndef R9VX_HOST_H
#define R9VX_HOST_H

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <string>

#include "r9vx.h"

/* Sets the calling thread's r9vx_last_error() text. */
void r9vx_set_last_error(const std::string &text);

namespace {

struct Problems {
    std::string text;
    int code = R9VX_OK;
    void add(int c, const char *fmt, ...) {
        char buf[256];
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(buf, sizeof buf, fmt, ap);
        va_end(ap);
        if (!text.empty()) text += "; ";
        text += buf;
        if (code == R9VX_OK) code = c;
    }
    int finish(const char *op) {
        if (code != R9VX_OK) r9vx_set_last_error(std::string(op) + ": " + text);
        return code;
    }
};

int hip_status(const char *op, int rc) {
    if (rc != 0)
        r9vx_set_last_error(std::string(op) + ": HIP error " + std::to_string(rc) + " (" +
                            hipGetErrorString((hipError_t)rc) + ")");
    return rc;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

/* Whether the two ranges share a byte (NULL: no range). */
bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && x < y + nb && y < x + na;
}

}  // namespace

#endif
