// group_rows.cu -- rows of a routed batch sorted by expert: a stable counting sort on the device, so that
// the ragged product that follows needs no word from the host.
//
//   offsets[e]  = number of rows with an id below e, e = 0 .. experts (ids outside [0, experts) count nowhere)
//   order[j]    = the row at sorted place j; rows of one expert keep their order; rows of no expert come last
//   position[r] = the sorted place of row r (the inverse of order)
//
// One cluster of CTAs does it in one launch: each warp owns a contiguous run of rows and counts its ids in
// shared memory; the counts of all warps of all CTAs, read over distributed shared memory, give every
// (warp, id) its first place; a second walk over the same run hands the places out, 32 rows at a time
// (__match_any_sync ranks equal ids among the lanes).  Whole numbers only, no atomics across CTAs: the
// result does not depend on timing.
#include <cooperative_groups.h>

#include "kernels.h"

namespace cg = cooperative_groups;

namespace smith {
namespace {

constexpr int kWarps = 16;            // x (1024 + 1) counters = 66 KB
constexpr int kThreads = kWarps * 32;
constexpr int kCluster = 8;

__global__ void __launch_bounds__(kThreads, 1) group_rows_kernel(const int* __restrict__ ids, int rows, int experts,
                                                                 int* __restrict__ offsets, int* __restrict__ order,
                                                                 int* __restrict__ position, int per_warp) {
  extern __shared__ int counts[];               // [kWarps][bins], then totals[bins], then scan scratch
  const int bins = experts + 1;                 // the last bin: rows of no expert
  int* totals = counts + kWarps * bins;
  int* warp_sum = totals + bins;                // [kWarps]
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < kWarps * bins; i += kThreads) counts[i] = 0;
  __syncthreads();

  const int64_t first = ((int64_t)rank * kWarps + warp) * per_warp;
  const int begin = (int)min(first, (int64_t)rows), end = (int)min(first + per_warp, (int64_t)rows);
  int* mine = counts + warp * bins;
  for (int r = begin + lane; r < end; r += 32) {
    int id = ids[r];
    if (id < 0 || id >= experts) id = experts;
    atomicAdd(&mine[id], 1);
  }
  __syncthreads();
  for (int b = tid; b < bins; b += kThreads) {  // counts of the warps before, within the CTA
    int sum = 0;
    for (int w = 0; w < kWarps; w++) {
      const int c = counts[w * bins + b];
      counts[w * bins + b] = sum;
      sum += c;
    }
    totals[b] = sum;
  }
  cluster.sync();
  // exclusive prefix over the bins of the totals of all CTAs; each thread a run of adjacent bins
  const int run = (bins + kThreads - 1) / kThreads;
  const int b0 = min(tid * run, bins), b1 = min(b0 + run, bins);
  int all = 0;
  for (int b = b0; b < b1; b++)
    for (int k = 0; k < ranks; k++) all += cluster.map_shared_rank(totals, k)[b];
  int incl = all;
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int start = incl - all;
  for (int w = 0; w < warp; w++) start += warp_sum[w];
  for (int b = b0; b < b1; b++) {
    int before = 0, sum = 0;
    for (int k = 0; k < ranks; k++) {
      const int c = cluster.map_shared_rank(totals, k)[b];
      if (k < rank) before += c;
      sum += c;
    }
    if (rank == 0) offsets[b] = start;          // offsets[experts] = where the rows of no expert begin
    for (int w = 0; w < kWarps; w++) counts[w * bins + b] += start + before;
    start += sum;
  }
  __syncthreads();

  for (int r0 = begin; r0 < end; r0 += 32) {
    const int r = r0 + lane;
    int id = -1;
    if (r < end) {
      id = ids[r];
      if (id < 0 || id >= experts) id = experts;
    }
    const unsigned same = __match_any_sync(0xffffffffu, id);
    if (id >= 0) {
      const int rank_here = __popc(same & ((1u << lane) - 1u));
      const int at = mine[id] + rank_here;
      position[r] = at;
      order[at] = r;
    }
    __syncwarp();
    if (id >= 0 && (same & ((1u << lane) - 1u)) == 0) mine[id] += __popc(same);
    __syncwarp();
  }
  cluster.sync();                               // no CTA leaves while another still reads its totals
}

}  // namespace

cudaError_t launch_group_rows(const int* ids, int64_t rows, int64_t experts, int* offsets, int* order, int* position,
                              cudaStream_t s) {
  if (rows < 0 || rows > 0x7FFFFFFF - 1024 || experts < 1 || experts > kInt8MaxExperts) return cudaErrorInvalidValue;
  const int bins = (int)experts + 1;
  const size_t smem = ((size_t)(kWarps + 1) * bins + kWarps) * 4;
  static PerDeviceFlag configured;
  bool* set = configured.here();
  if (!set) return cudaErrorInvalidDevice;
  if (!*set) {
    const cudaError_t e = cudaFuncSetAttribute(group_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    if (e != cudaSuccess) return e;
    *set = true;
  }
  int64_t per_warp = (rows + kCluster * kWarps - 1) / (kCluster * kWarps);
  per_warp = (per_warp + 31) / 32 * 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kCluster, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, group_rows_kernel, ids, (int)rows, (int)experts, offsets, order, position, (int)per_warp);
}

}  // namespace smith
