#include "launch_info.h"

#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <tuple>

namespace mmf {

namespace {

std::mutex lock;
std::map<std::pair<const void*, int>, int> allowed;                     // (kernel, device): bytes
std::map<std::tuple<const void*, int, int, int>, int> resident;         // (kernel, device, block, smem): blocks
std::map<std::tuple<const void*, int, int, int, int>, int> clusters;    // (the same and blocks a cluster): clusters

void check(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("mmf: preparing a kernel: ") + cudaGetErrorString(e));
}

int current_device() {
  int device = 0;
  check(cudaGetDevice(&device));
  return device;
}

void allow(const void* kernel, int device, int smem, bool carveout) {
  const auto key = std::make_pair(kernel, device);
  const auto it = allowed.find(key);
  if (it != allowed.end() && it->second >= smem) return;
  check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (carveout)
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  allowed[key] = smem;
}

}  // namespace

void allow_shared(const void* kernel, int smem, bool carveout) {
  const int device = current_device();
  std::lock_guard<std::mutex> hold(lock);
  allow(kernel, device, smem, carveout);
}

int resident_blocks(const void* kernel, int block, int smem) {
  const int device = current_device();
  std::lock_guard<std::mutex> hold(lock);
  const auto key = std::make_tuple(kernel, device, block, smem);
  const auto it = resident.find(key);
  if (it != resident.end()) return it->second;
  allow(kernel, device, smem, false);
  int blocks = 0;
  check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, block, static_cast<size_t>(smem)));
  if (blocks < 1) throw std::runtime_error("mmf: preparing a kernel: no block of it fits an SM");
  return resident[key] = blocks;
}

int resident_clusters(const void* kernel, int block, int smem, int blocks) {
  const int device = current_device();
  std::lock_guard<std::mutex> hold(lock);
  const auto key = std::make_tuple(kernel, device, block, smem, blocks);
  const auto it = clusters.find(key);
  if (it != clusters.end()) return it->second;
  allow(kernel, device, smem, false);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(1024, static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = attr.val.clusterDim.z = 1;
  attr.val.clusterDim.y = static_cast<unsigned>(blocks);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  check(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
  if (n < 1) throw std::runtime_error("mmf: preparing a kernel: no cluster of it fits the device");
  return clusters[key] = n;
}

}  // namespace mmf
