/*
 * g4s_host.h -- what the entry points of the beam search, the page cache and
 * the 8-bit cache share on the host: handles, devices, workspaces and the
 * check of arrays against each other.
 */
#ifndef G4S_HOST_H
#define G4S_HOST_H

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "gemma4_sampler.h"

#define G4S_API extern "C" __attribute__((visibility("default")))

namespace g4s {

struct Handle {
    int device = 0;
    hipStream_t stream = nullptr;
    char err[512] = "";
};

inline int fail_in(char (&buf)[512], int code, const char* fmt, va_list ap)
{
    vsnprintf(buf, sizeof(buf), fmt, ap);
    return code;
}

/* The handle's device is current while a call works with it. */
class DeviceGuard {
public:
    explicit DeviceGuard(int device)
    {
        if (hipGetDevice(&old_) != hipSuccess) old_ = device;
        if (old_ != device)
            ok_ = hipSetDevice(device) == hipSuccess;
        else
            old_ = -1;
    }
    ~DeviceGuard()
    {
        if (old_ >= 0) (void)hipSetDevice(old_);
    }
    bool ok() const { return ok_; }

private:
    int old_ = -1;
    bool ok_ = true;
};

/* The current device, if the library runs on it: G4S_OK, or what `refuse` makes of a
 * code and a printf message. */
template <typename F>
int pick_device(F refuse, int* device, int* ncu = nullptr)
{
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n < 1)
        return refuse(G4S_ERR_NO_DEVICE, "no HIP device visible");
    hipDeviceProp_t prop;
    if (hipGetDevice(device) != hipSuccess ||
        hipGetDeviceProperties(&prop, *device) != hipSuccess)
        return refuse(G4S_ERR_NO_DEVICE, "the current HIP device is not usable");
    if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
        return refuse(G4S_ERR_NO_DEVICE, "device %d is %s; this library targets gfx950", *device,
                      prop.gcnArchName);
    if (ncu) *ncu = prop.multiProcessorCount;
    return G4S_OK;
}

inline bool overlap(const void* a, int64_t na, const void* b, int64_t nb)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

/* An array of a call; NULL ones overlap nothing. */
struct Span {
    const char* name;
    const void* at;
    int64_t bytes;
};
inline bool overlap(const Span& a, const Span& b)
{
    return a.at && b.at && overlap(a.at, a.bytes, b.at, b.bytes);
}

/* Parts of one allocation, each on a 256-byte boundary. */
class Carver {
public:
    template <typename T>
    void add(T** p, size_t count)
    {
        if (base_) *p = reinterpret_cast<T*>(base_ + used_);
        used_ += (count * sizeof(T) + 255) & ~(size_t)255;
    }
    size_t used() const { return used_; }
    void start(void* base)
    {
        base_ = static_cast<char*>(base);
        used_ = 0;
    }

private:
    char* base_ = nullptr;
    size_t used_ = 0;
};

}  // namespace g4s

#endif
