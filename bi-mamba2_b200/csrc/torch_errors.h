// A library status as a C++ exception; it becomes ssd._cabi.BissdError in Python.
#pragma once
#include <stdexcept>
#include <string>

#include "../../include/bissd.h"

struct BissdError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

inline void bissd_check(int rc) {
    if (rc == BISSD_OK) return;
    const char *cuda = bissd_last_cuda_error();
    std::string msg = "libbissd error " + std::to_string(rc) + ": " + bissd_strerror(rc);
    if (cuda && cuda[0]) msg += std::string(" [") + cuda + "]";
    throw BissdError(msg);
}

// Tests and debugging: a synchronising read of the device status word after every pass.
inline void bissd_check_device_status(bool on, const void *ws, void *stream) {
    if (!on) return;
    int st = 0;
    bissd_check(bissd_read_status(ws, stream, &st));
    if (st != 0)
        throw BissdError("libbissd device status " + std::to_string(st) + ": a device-side wait ran out; results are invalid");
}
