// The runtime's side of a kernel launch, for programs that run an entry point's host code without a device:
// a launch is recorded (kernel, grid, block, its arguments' addresses) and nothing runs.  Include it
// before the source that is under test, and link no HIP runtime.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <functional>

namespace launches {

struct Config {
  dim3 grid, block;
  size_t shared;
  hipStream_t stream;
};
inline Config pending;
// what a launch is given to: (kernel, grid, block, arguments)
inline std::function<void(const void*, const dim3&, const dim3&, void**)> seen;

}  // namespace launches

extern "C" {
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t stream) {
  launches::pending = {grid, block, shared, stream};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
  *grid = launches::pending.grid;
  *block = launches::pending.block;
  *shared = launches::pending.shared;
  *stream = launches::pending.stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void** args, size_t, hipStream_t) {
  launches::seen(f, grid, block, args);
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned int, void*, void*, void*, void*, int*) {}
void __hipRegisterVar(void**, void*, char*, const char*, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void**) {}
}
