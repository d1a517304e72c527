// int8_gemm.cu -- C = scale_a[m] * scale_w[n] * (codes_a x codes_w) on the 8-bit integer tensor cores,
// for one weight matrix or for rows sorted by expert with a matrix each.
//
//   c[m, n] = (sum_k ca[m, k] * cw[n, k]) * sa[m] * sw[n],   s = max / 127
// The sum is a whole number below 127^2 * 131072 < 2^31: s32 accumulators hold it exactly.  The scales
// are applied in f32, f32(sum) * sa * sw in that order (three roundings, and the scales' own), where both
// lie in [2^-60, 2^60] or are 0: no product on the way then leaves f32's normal range unless c does.  For
// other scales that element is formed in f64 and rounded once.  f16 results round the f32 value.
//
// The weights are the MMA's first operand (128 channels are the 128 lanes of the accumulator), the
// tokens its second: a tile takes 16 to 256 tokens, so one token wastes little, and lane = channel lets
// the epilogue store each token's 32 channels per warp as one contiguous segment without a transpose.
//
// One CTA per tile of 128 channels x BT tokens: a producer thread (one bulk copy of the packed 16 KB
// weight block and one tensor-map box of token codes per 128 k), an MMA thread, four epilogue warps.
// Every mbarrier wait is time-bounded (pipeline.cuh).
#include <cuda.h>
#include <cuda_fp16.h>

#include "int8_gemm.cuh"
#include "kernels.h"
#include "pipeline.cuh"
#include "qgemv_common.cuh"
#include "tcgen05.cuh"

namespace smith {
namespace {

constexpr int kThreads = 6 * 32;
constexpr int kWTile = 16384;         // 128 channels x 128 k
constexpr int kMaxStages = 12;

struct Params {
  const uint8_t* w;
  const float* w_max;                 // [experts][n_tiles * 128]
  const float* a_max;                 // [rows]
  const int* offsets;                 // null: one group of all rows; else [experts + 1]
  const int* order;                   // null, or the row of C for each sorted row
  void* C;
  int64_t ldc;
  int rows, N, experts;
  int n_tiles, k_slabs;
  int BT;                             // tokens per tile
  int stages, stage_bytes, tmem_cols;
  int out_f16;
  uint32_t idesc;
  int* status;
};

// Group boundaries come from device memory: clamped, so that nothing they hold leads outside the rows.
__device__ __forceinline__ void group_range(const Params& p, int e, int& first, int& count) {
  if (!p.offsets) {
    first = 0, count = p.rows;
    return;
  }
  first = min(max(p.offsets[e], 0), p.rows);
  count = min(max(p.offsets[e + 1], first), p.rows) - first;
}

__device__ __forceinline__ float scale_of(float most) {
  return __float_as_uint(most) >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __fdiv_rn(most, 127.f);
}
__device__ __forceinline__ bool plain_scale(float s) {
  return !(fabsf(s) < 0x1p-60f || fabsf(s) > 0x1p60f) || s == 0.f;      // a NaN is as good in f32
}
__device__ __forceinline__ float scaled(int sum, float sa, float sw, float a_max, float w_max) {
  if (plain_scale(sa) && plain_scale(sw)) return (float)sum * sa * sw;
  return (float)((double)sum * ((double)a_max / 127.0) * ((double)w_max / 127.0));
}

__global__ void __launch_bounds__(kThreads, 1) int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_ready = empty + kMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_ready + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* found = reinterpret_cast<int*>(tmem_slot + 2);      // expert, first row, rows of the tile
  uint8_t* tiles = smem + 1024;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nt = blockIdx.y;

  if (tid == 0) {
    for (int s = 0; s < kMaxStages; s++) mbar_init(smem_u32(&full[s]), 1), mbar_init(smem_u32(&empty[s]), 1);
    mbar_init(smem_u32(acc_ready), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    // which expert and which of its token tiles
    int before = 0, x = blockIdx.x;
    if (lane == 0) found[0] = -1;
    __syncwarp();
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      int first = 0, count = 0;
      if (e0 + lane < p.experts) group_range(p, e0 + lane, first, count);
      const int t = (count + p.BT - 1) / p.BT;
      int incl = t;
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      const int lo = before + incl - t;
      if (x >= lo && x < lo + t) {
        found[0] = e0 + lane;
        found[1] = first + (x - lo) * p.BT;
        found[2] = min(count - (x - lo) * p.BT, p.BT);
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      if (x < before) break;
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), (uint32_t)p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int expert = found[0], row0 = found[1], rows = found[2];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (expert >= 0) {
    if (warp == 0) {
      if (lane == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const uint8_t* src = p.w + ((size_t)expert * p.n_tiles + nt) * (size_t)p.k_slabs * kWTile;
        int s = 0;
        uint32_t par = 0;
        for (int ks = 0; ks < p.k_slabs; ks++) {
          if (ks >= p.stages && !mbar_wait(smem_u32(&empty[s]), par ^ 1u, abort_flag, p.status)) break;
          const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(tiles) + (uint32_t)(s * p.stage_bytes);
          mbar_expect_tx(bar, (uint32_t)p.stage_bytes);
          bulk_load_plain(dst, src + (size_t)ks * kWTile, kWTile, bar);
          tma_load_2d(dst + kWTile, &tmap, ks * 128, row0, bar);   // rows beyond the last are zeros and count
          if (++s == p.stages) s = 0, par ^= 1u;
        }
      }
    } else if (warp == 1) {
      if (lane == 0) {
        const uint64_t desc0 = smem_desc_sw128(smem_u32(tiles));
        const uint32_t lo0 = (uint32_t)desc0, hi = (uint32_t)(desc0 >> 32);
        int s = 0;
        uint32_t par = 0;
        bool ok = true;
        for (int ks = 0; ks < p.k_slabs; ks++) {
          ok = mbar_wait(smem_u32(&full[s]), par, abort_flag, p.status);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = lo0 + (uint32_t)((s * p.stage_bytes) >> 4);
          umma_i8_kblock(tmem, a_lo, a_lo + (kWTile >> 4), hi, p.idesc, ks > 0 ? 1u : 0u);
          umma_commit(smem_u32(&empty[s]));
          if (++s == p.stages) s = 0, par ^= 1u;
        }
        if (ok) umma_commit(smem_u32(acc_ready));
      }
    } else {
      asm volatile("griddepcontrol.wait;" ::: "memory");       // a_max is the previous launch's
      const bool got = __all_sync(0xffffffffu, mbar_wait(smem_u32(acc_ready), 0, abort_flag, p.status));
      tc_fence_after();
      if (got) {
        const int q = warp & 3;
        const int n = nt * 128 + q * 32 + lane;
        float w_max = p.w_max[(size_t)expert * p.n_tiles * 128 + n];
        const float sw = scale_of(w_max);
        if (sw != sw) w_max = sw;
        for (int c = 0; c < rows; c += 32) {
          uint32_t r[32];
          tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
          tmem_ld_wait();
          float a_max = 0.f;
          int to = -1;
          if (c + lane < rows) {
            const int row = row0 + c + lane;
            a_max = p.a_max[row];
            to = p.order ? p.order[row] : row;
            if (to >= p.rows) to = -1;
          }
          const float sa = scale_of(a_max);
          const bool plain = __all_sync(0xffffffffu, plain_scale(sa) && plain_scale(sw));
#pragma unroll
          for (int i = 0; i < 32; i++) {
            const int at = __shfl_sync(0xffffffffu, to, i);
            const float si = __shfl_sync(0xffffffffu, sa, i);
            const float v = plain ? (float)(int)r[i] * si * sw
                                  : scaled((int)r[i], si, sw, __shfl_sync(0xffffffffu, a_max, i), w_max);
            if (at >= 0 && n < p.N) {
              if (p.out_f16) static_cast<__half*>(p.C)[at * p.ldc + n] = __float2half_rn(v);
              else static_cast<float*>(p.C)[at * p.ldc + n] = v;
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
  }
}

bool encode_codes(CUtensorMap* map, const void* base, int64_t kp, int64_t rows, int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)kp, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)kp};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace

size_t int8_gemm_workspace_bytes(int64_t rows, int64_t K) {
  return align_up((size_t)rows * align_up((size_t)K, 128), 1024) + align_up((size_t)rows * 4, 256);
}

cudaError_t launch_int8_gemm(const Int8Gemm& g, Workspace ws, cudaStream_t s) {
  if (!ws.ptr || ws.bytes < int8_gemm_workspace_bytes(g.rows, g.K)) return cudaErrorInvalidValue;
  const int8_layout l = int8_weight_layout(g.K, g.N, g.experts);
  uint8_t* codes = static_cast<uint8_t*>(ws.ptr);
  const int64_t kp = l.k_slabs * 128;
  float* a_max = reinterpret_cast<float*>(codes + align_up((size_t)g.rows * kp, 1024));
  cudaError_t e = launch_int8_rows(g.dtype, g.A, g.position ? g.rows / g.fan : g.rows, g.lda, g.K, g.position, g.fan, g.rows,
                                   codes, a_max, s);
  if (e != cudaSuccess) return e;

  // tokens per tile: the power of two at or above the rows of a group, on average
  const int64_t mean = (g.rows + g.experts - 1) / g.experts;
  int bt = 16;
  while (bt < mean && bt < 256) bt <<= 1;
  CUtensorMap map;
  if (!encode_codes(&map, codes, kp, g.rows, bt)) return cudaErrorInvalidValue;
  Params p{};
  p.w = static_cast<const uint8_t*>(g.W);
  p.w_max = reinterpret_cast<const float*>(p.w + l.code_bytes);
  p.a_max = a_max;
  p.offsets = g.offsets, p.order = g.order, p.C = g.C, p.ldc = g.ldc;
  p.rows = (int)g.rows, p.N = (int)g.N, p.experts = (int)g.experts;
  p.n_tiles = (int)l.n_tiles, p.k_slabs = (int)l.k_slabs, p.BT = bt;
  p.stage_bytes = kWTile + bt * 128;
  p.stages = (226 * 1024 - 1024) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.tmem_cols = bt < 32 ? 32 : bt;
  p.out_f16 = g.dtype == kDenseF16;
  // tcgen05.mma kind::i8 instruction descriptor: [4,6) D = s32 (2); [7,10) A and [10,13) B signed 8-bit (1);
  // both operands K-major; [17,23) N >> 3; [24,29) M >> 4
  p.idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(bt >> 3) << 17) | (8u << 24);
  p.status = kernel_status_ptr();
  if (!p.status) return cudaErrorUnknown;
  static PerDeviceFlag configured;
  bool* set = configured.here();
  if (!set) return cudaErrorInvalidDevice;
  if (!*set) {
    e = cudaFuncSetAttribute(int8_gemm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    *set = true;
  }
  int64_t token_tiles = (g.rows + bt - 1) / bt;
  if (g.offsets) token_tiles += g.experts;        // at most: each group's last tile is partly empty
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)token_tiles, (unsigned)l.n_tiles), cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 1024 + (size_t)p.stages * p.stage_bytes, cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, int8_gemm_kernel, map, p);
}

}  // namespace smith
