// How the library launches its kernels (included by its translation units).
#pragma once

#include <cuda_runtime.h>

// Opt-in limits and caches are kept per device: the library may be used on every GPU of a box from one process.
#define PYLO_MAX_DEVICES 64
inline int g_sm_count[PYLO_MAX_DEVICES] = {0};
inline int sm_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= PYLO_MAX_DEVICES) return 148;
  if (g_sm_count[dev] == 0) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    g_sm_count[dev] = n > 0 ? n : 148;
  }
  return g_sm_count[dev];
}
inline int grid_for(int n_items, int ctas_per_sm) {
  const int cap = sm_count() * ctas_per_sm;
  return n_items < cap ? n_items : cap;
}
inline int launch_status() { return (int)cudaGetLastError(); }

// Every kernel of this library is launched so that it may become resident while its predecessor in the stream drains
// (programmatic dependent launch) and waits in pdl_begin() until that one is complete.  A step is a chain of small launches;
// on a small model the gaps between them are as long as the kernels (AdafacLO over a 118 K MLP: 47.5 -> 38.8 us per step).
// On large ones there is nothing to gain (GPT-2-medium shapes: 0.7 % slower with it), so a step of more than 134 M elements
// launches plainly: PlainLaunches says so for the calls of one scope on one host thread.
inline thread_local bool t_plain_launches = false;
struct PlainLaunches {
  bool before;
  explicit PlainLaunches(int n_tiles) : before(t_plain_launches) { t_plain_launches = before || n_tiles > 8192; }
  ~PlainLaunches() { t_plain_launches = before; }
};
// The SMs' memory is split between L1 cache and shared memory anew only when they are idle, which programmatic launches never
// let them be: the kernels after one with a large share of shared memory would run with what L1 it left (the apply sweep of
// 6 x 4096 x 4096 VeLO parameters: 921 us after the state sweep's ring, 755 us without).  Such a kernel has itself and the next
// launch of its thread made plainly.
inline thread_local bool t_plain_next = false;
// For the launches of one scope: kernels that stream through memory and do not mind.  What they are followed by still does.
struct AnyCache {
  bool next;
  AnyCache() : next(t_plain_next) { t_plain_next = false; }
  ~AnyCache() { t_plain_next = next; }
};
template <class... P, class... A>
static void launch_clusters(void (*kernel)(P...), dim3 grid, dim3 block, int cluster, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (!t_plain_launches && !t_plain_next) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  t_plain_next = false;
  if (cluster >= 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
template <class... P, class... A>
static void launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
  launch_clusters(kernel, grid, block, 0, smem, stream, static_cast<A&&>(args)...);
}

// Opt a kernel in to more than 48 KB of dynamic shared memory, once per device (the attribute belongs to the
// device's copy of the function); flags[] is the caller's per-kernel record.
template <class K>
static int allow_dynamic_smem(K kernel, int bytes, bool (&flags)[PYLO_MAX_DEVICES]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 0 && dev < PYLO_MAX_DEVICES && flags[dev]) return 0;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 0 && dev < PYLO_MAX_DEVICES) flags[dev] = true;
  return 0;
}

// Clusters of 2, 4 or 8 CTAs that run at once (of single CTAs for 1): not every group of SMs that a cluster has to stay in holds a multiple of it.
template <auto KERNEL>
static int active_clusters(int threads, int cluster, size_t smem) {
  static int known[PYLO_MAX_DEVICES][4] = {};
  static size_t known_smem[PYLO_MAX_DEVICES][4] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const int at = cluster == 1 ? 0 : cluster == 2 ? 1 : cluster == 4 ? 2 : 3;
  const bool kept = dev >= 0 && dev < PYLO_MAX_DEVICES;
  if (kept && known[dev][at] && known_smem[dev][at] == smem) return known[dev][at];
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = cluster;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = sm_count() / cluster > 0 ? sm_count() / cluster : 1;
  }
  if (kept) { known[dev][at] = n; known_smem[dev][at] = smem; }
  return n;
}

#define CHECK_ARG(cond) \
  do {                  \
    if (!(cond)) return -1; \
  } while (0)
