// A stand-in for the HIP runtime in front of libgpumon_diag.so (LD_PRELOAD), so that the CPU tests see what its entry points refuse and
// what they would launch: two devices, the current one 0; memory from 4 GiB on lies on device 1; a launch prints its grid
// and block and reaches no GPU.
// build: g++ -shared -fPIC -D__HIP_PLATFORM_AMD__ -I/opt/rocm/include tests/stubs/hip_stub.cc -o libhip_stub.so
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstring>

extern "C" {
hipError_t hipGetDeviceCount(int* n) { return *n = 2, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t* d) { return *d = 0, hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* at, const void* p) {
  memset(at, 0, sizeof *at);
  at->type = hipMemoryTypeDevice;
  at->device = (size_t)p >= (1ull << 32);
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
// what a <<<grid, block>>> begins with; anything but success leaves the kernel out
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t) {
  printf("launch %u %u %u x %u %u %u\n", grid.x, grid.y, grid.z, block.x, block.y, block.z);
  fflush(stdout);
  return hipErrorNotReady;
}
}
