// grant_smem (mvcc_b200/csrc/moe_common.cuh) from two host threads, over stand-ins for the runtime's calls that keep the
// attribute here and let the larger request linger between setting it and returning.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

#define cudaGetDevice stand_in_get_device
#define cudaFuncSetAttribute stand_in_set_attribute
static cudaError_t cudaGetDevice(int* d);
static cudaError_t cudaFuncSetAttribute(const void* kern, cudaFuncAttribute what, int value);
#include "../../mvcc_b200/csrc/moe_common.cuh"

static std::atomic<int> attribute{0}, calls{0};
static std::atomic<bool> large_set{false}, small_done{false};

static cudaError_t cudaGetDevice(int* d) {
  *d = 0;
  return cudaSuccess;
}
static cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int value) {
  ++calls;
  attribute = value;
  if (value > 64 * 1024) {
    large_set = true;
    for (int i = 0; i < 200 && !small_done; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
  }
  return cudaSuccess;
}

int main() {
  static moe::SmemGrant g;
  const size_t large = 88 * 1024, floor_bytes = 64 * 1024;
  std::thread a([&] { moe::grant_smem(nullptr, large, floor_bytes, g); });
  while (!large_set) std::this_thread::yield();
  std::thread b([&] {
    moe::grant_smem(nullptr, 1024, floor_bytes, g);
    small_done = true;
  });
  a.join();
  b.join();
  moe::grant_smem(nullptr, large, floor_bytes, g);  // what a later launch of the large size relies on
  std::printf("attribute %d after %d calls\n", attribute.load(), calls.load());
  return attribute.load() >= (int)large ? 0 : 1;
}
