// ops.cu -- the operators' handle (pt_b200_ops_*).
#include <new>

#include "linear_tc.cuh"

using namespace ptb;

extern "C" pt_b200_ops *pt_b200_ops_create(int device) {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n) {
    cudaGetLastError();
    set_error("pt_b200_ops_create: device %d out of range (%d present; there is no CPU path)", device, n);
    return nullptr;
  }
  DeviceScope on(device);
  cudaDeviceProp prop;
  if (!on.ok || cudaGetDeviceProperties(&prop, device) != cudaSuccess) {
    set_error("pt_b200_ops_create: device %d cannot be used", device);
    return nullptr;
  }
  if (prop.major != 10 || prop.minor != 0) {
    set_error("pt_b200_ops_create: device %d is sm_%d%d; this library is built for sm_100a (B200) only",
              device, prop.major, prop.minor);
    return nullptr;
  }
  uint32_t *gerr = nullptr;
  if (cudaMalloc(&gerr, 256) != cudaSuccess || cudaMemset(gerr, 0, 256) != cudaSuccess) {
    cudaFree(gerr);
    set_error("pt_b200_ops_create: out of device memory");
    return nullptr;
  }
  pt_b200_ops *h = new (std::nothrow) pt_b200_ops{device, prop.multiProcessorCount, gerr, {}};
  if (!h || tc_setup(h)) {
    cudaFree(gerr);
    delete h;
    return nullptr;
  }
  return h;
}

extern "C" void pt_b200_ops_destroy(pt_b200_ops *h) {
  if (!h) return;
  DeviceScope on(h->device);
  cudaFree(h->gerr);
  delete h;
}

extern "C" int pt_b200_ops_sync(pt_b200_ops *h, void *stream) {
  PTB_REQUIRE(h, "pt_b200_ops_sync: NULL handle");
  DeviceScope on(h->device);
  PTB_REQUIRE(on.ok, "pt_b200_ops_sync: device %d cannot be used", h->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (wait_stream(st)) return -1;
  uint32_t err = 0;
  PTB_CUDA(cudaMemcpyAsync(&err, h->gerr, 4, cudaMemcpyDeviceToHost, st));
  if (wait_stream(st)) return -1;
  if (err) {
    PTB_CUDA(cudaMemsetAsync(h->gerr, 0, 4, st));
    set_error("pt_b200_ops_sync: device error word 0x%x (a bounded wait gave up)", err);
    return -1;
  }
  return 0;
}
