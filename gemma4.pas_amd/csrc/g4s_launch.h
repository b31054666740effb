/*
 * g4s_launch.h -- a kernel launch that reports itself.
 *
 * hipGetLastError() after a launch also gives what an earlier call of the same thread
 * left there, the caller's own failures among them: a launch that is
 * under way would be reported as failed, and repeating a move in place is
 * another move.
 */
#ifndef G4S_LAUNCH_H
#define G4S_LAUNCH_H

#include <hip/hip_runtime.h>

#include <type_traits>

namespace g4s {

template <typename... P>
hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t stream,
                  std::type_identity_t<P>... args)
{
    void* at[] = {const_cast<void*>(static_cast<const void*>(&args))...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, at, lds, stream);
}

}  // namespace g4s

#endif
