// group_rows.cu -- rows of a routed batch sorted by expert: a stable counting sort on the device, so that
// the ragged product that follows needs no word from the host.
//
//   offsets[e]  = number of rows with an id below e, e = 0 .. experts (ids outside [0, experts) count nowhere)
//   order[j]    = the row at sorted place j; rows of one expert keep their order; rows of no expert come last
//   position[r] = the sorted place of row r (the inverse of order)
//
// Each warp owns a contiguous run of rows and counts its ids in shared memory; the counts of all warps that
// come before it, and of all smaller ids, give every (warp, id) its first place; a second walk over the run
// hands the places out, 32 rows at a time (__match_any_sync ranks equal ids among the lanes).  Whole
// numbers only, no atomics across CTAs: the result does not depend on timing.
//
// Few rows are one CTA's work.  More are spread over half the SMs in two launches: one counts the ids of each
// CTA's run into scratch, the other adds the counts of all runs up and hands out places.  All of it is
// latency: 256 rows of 64 experts 2.5 us, 4096 rows 6.1 us by one CTA and 5.1 by several, 262144 rows of 256
// experts 10.5 us (16 warps per CTA 11.6, all SMs 16.2, a cluster of 8 CTAs that exchanged counts over
// distributed shared memory 40), of 1024 experts 17.8 us (16 warps 28.6).
#include "kernels.h"

namespace smith {
namespace {

constexpr int kFewWarps = 16, kManyWarps = 32;      // 32 warps x (1024 + 1) counters = 131 KB
constexpr int kOneCta = 2560;         // up to so many rows one CTA does it alone
constexpr int kManyRows = 32768;      // from there on kManyWarps per CTA

__device__ __forceinline__ int bin_of(const int* ids, int r, int experts) {
  const int id = ids[r];
  return id < 0 || id >= experts ? experts : id;
}

struct Run {
  int begin, end;
  __device__ Run(int64_t first, int length, int rows)
      : begin((int)min(first, (int64_t)rows)), end((int)min(first + length, (int64_t)rows)) {}
};

__host__ __device__ constexpr int padded(int bins) { return (bins + 3) / 4 * 4; }

// counts[block][bin] of each block's rows, rows of padded(bins)
template <int warps>
__global__ void __launch_bounds__(warps * 32) group_count_kernel(const int* ids, int rows, int experts, int per_warp, int* block_counts) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ int counts[];               // [bins]
  constexpr int threads = warps * 32;
  const int bins = experts + 1;
  for (int i = threadIdx.x; i < padded(bins); i += threads) counts[i] = 0;
  __syncthreads();
  const Run run((int64_t)blockIdx.x * warps * per_warp, warps * per_warp, rows);
  for (int r = run.begin + threadIdx.x; r < run.end; r += threads) atomicAdd(&counts[bin_of(ids, r, experts)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < padded(bins); i += threads) block_counts[(int64_t)blockIdx.x * padded(bins) + i] = counts[i];
}

// block_counts null: the one block's own counts are all there are
template <int warps>
__global__ void __launch_bounds__(warps * 32, 1) group_place_kernel(const int* ids, int rows, int experts, int* offsets, int* order,
                                                                  int* position, int per_warp, const int* block_counts) {
  extern __shared__ int counts[];               // [warps][bins], then before[bins], all[bins]
  constexpr int threads = warps * 32;
  const int bins = experts + 1;
  int* before = counts + warps * bins;          // rows of the bin in the blocks before this one
  int* all = before + bins;                     // in all blocks; then the bin's first place
  __shared__ int warp_sum[warps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < (warps + 2) * bins; i += threads) counts[i] = 0;
  __syncthreads();
  const Run run(((int64_t)blockIdx.x * warps + warp) * per_warp, per_warp, rows);
  int* mine = counts + warp * bins;
  for (int r = run.begin + lane; r < run.end; r += 32) atomicAdd(&mine[bin_of(ids, r, experts)], 1);
  if (block_counts) {
    // only the counts come from the launch before; ids were there before that one began
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // four bins to a load; as many threads as fit share the blocks of a column
    const int columns = padded(bins) / 4, parts = threads / columns, part = tid / columns, column = tid - part * columns;
    if (part < parts) {
      const int4* from = reinterpret_cast<const int4*>(block_counts) + column;
      int4 sum = make_int4(0, 0, 0, 0), head = sum;
#pragma unroll 8
      for (int k = part; k < (int)gridDim.x; k += parts) {
        const int4 c = __ldcg(from + (int64_t)k * columns);
        sum.x += c.x, sum.y += c.y, sum.z += c.z, sum.w += c.w;
        if (k < (int)blockIdx.x) head.x += c.x, head.y += c.y, head.z += c.z, head.w += c.w;
      }
      const int s[4] = {sum.x, sum.y, sum.z, sum.w}, h[4] = {head.x, head.y, head.z, head.w};
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (4 * column + j < bins) atomicAdd(&all[4 * column + j], s[j]), atomicAdd(&before[4 * column + j], h[j]);
    }
  }
  __syncthreads();
  for (int b = tid; b < bins; b += threads) {  // rows of the bin in the warps before, within the block
    int sum = 0;
    for (int w = 0; w < warps; w++) {
      const int c = counts[w * bins + b];
      counts[w * bins + b] = sum;
      sum += c;
    }
    if (!block_counts) all[b] = sum;
  }
  __syncthreads();
  // exclusive prefix over the bins; each thread a run of adjacent bins
  const int length = (bins + threads - 1) / threads;
  const int b0 = min(tid * length, bins), b1 = min(b0 + length, bins);
  int own = 0;
  for (int b = b0; b < b1; b++) own += all[b];
  int incl = own;
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int start = incl - own;
  for (int w = 0; w < warp; w++) start += warp_sum[w];
  for (int b = b0; b < b1; b++) {
    if (blockIdx.x == 0) offsets[b] = start;    // offsets[experts] = where the rows of no expert begin
    before[b] += start;
    start += all[b];
  }
  __syncthreads();

  for (int r0 = run.begin; r0 < run.end; r0 += 32) {
    const int r = r0 + lane;
    const int id = r < run.end ? bin_of(ids, r, experts) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    const unsigned lower = same & ((1u << lane) - 1u);
    if (id >= 0) {
      const int at = before[id] + mine[id] + __popc(lower);
      position[r] = at;
      order[at] = r;
    }
    __syncwarp();
    if (id >= 0 && lower == 0) mine[id] += __popc(same);
    __syncwarp();
  }
}

int place_blocks(int64_t rows) {
  if (rows <= kOneCta) return 1;
  const int64_t want = (rows + 1023) / 1024, most = device_sm_count() / 2;   // every block reads all blocks' counts
  return (int)(want < most ? want : most);
}

}  // namespace

size_t group_rows_workspace_bytes(int64_t rows, int64_t experts) {
  const int blocks = place_blocks(rows);
  return blocks > 1 ? (size_t)blocks * padded((int)experts + 1) * 4 : 0;
}

cudaError_t launch_group_rows(const int* ids, int64_t rows, int64_t experts, int* offsets, int* order, int* position,
                              Workspace ws, cudaStream_t s) {
  if (rows < 0 || rows > 0x7FFFFFFF - 1024 || experts < 1 || experts > kInt8MaxExperts) return cudaErrorInvalidValue;
  if (ws.bytes < group_rows_workspace_bytes(rows, experts)) return cudaErrorInvalidValue;
  const int bins = (int)experts + 1, blocks = place_blocks(rows);
  const bool many = rows > kManyRows;
  const int per_block = many ? kManyWarps : kFewWarps;
  const size_t smem = (size_t)(per_block + 2) * bins * 4;
  const auto count = many ? group_count_kernel<kManyWarps> : group_count_kernel<kFewWarps>;
  const auto place = many ? group_place_kernel<kManyWarps> : group_place_kernel<kFewWarps>;
  static PerDeviceFlag configured;
  bool* set = configured.here();
  if (!set) return cudaErrorInvalidDevice;
  if (!*set) {
    for (const auto k : {group_place_kernel<kFewWarps>, group_place_kernel<kManyWarps>}) {
      const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
      if (e != cudaSuccess) return e;
    }
    *set = true;
  }
  const int64_t warps = (int64_t)blocks * per_block;
  const int per_warp = (int)(((rows + warps - 1) / warps + 31) / 32 * 32);
  int* block_counts = blocks > 1 ? static_cast<int*>(ws.ptr) : nullptr;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks), cfg.blockDim = dim3((unsigned)per_block * 32), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr, cfg.numAttrs = 0;
  if (blocks > 1) {
    count<<<blocks, per_block * 32, (size_t)padded(bins) * 4, s>>>(ids, (int)rows, (int)experts, per_warp, block_counts);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cfg.numAttrs = 1;
  }
  count_launch();
  return cudaLaunchKernelEx(&cfg, place, ids, (int)rows, (int)experts, offsets, order, position, per_warp,
                            (const int*)block_counts);
}

}  // namespace smith
