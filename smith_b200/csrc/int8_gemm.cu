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
// One persistent launch.  A tile is 128 channels (a CTA pair: 256) by BT tokens of one group, a unit one
// slab of 128 k of a tile; tiles are ordered with tokens fastest, then channels, then groups, so weights
// come from HBM once and the token codes stay in L2.  The units of all tiles are dealt to the workers
// (CTAs or pairs) in equal contiguous runs where whole tiles would leave workers idle; a tile that two or
// more workers share is joined by the one that finishes last: the others leave their s32 partial sums in
// a slot of scratch and count themselves on a counter (zeroed by the launch that makes the codes).  Whole
// numbers add in any order, so the result does not depend on which one is last, and nobody waits.
//
//   warp 0     producer: one copy of the packed 16 KB weight block and one box of token codes per unit
//   warp 1     MMA issuer; two accumulators in tensor memory, so the next tile runs during an epilogue
//   warps 2-5  epilogue
// Every mbarrier wait is time-bounded (pipeline.cuh); on a give-up the CTA waits (bounded) for its copies
// and MMAs in flight, frees its tensor memory and leaves the status word set.
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
constexpr int kHeader = 1536;         // barriers; the group lists follow
constexpr int kSplitCost = 8;         // units of time that joining a shared tile costs (see `share` below)
constexpr int kMinUnits = 4;          // fewest units per worker

struct Params {
  const uint8_t* w;
  const float* w_max;                 // [experts][n_tiles * 128]
  const float* a_max;                 // [rows]
  const int* offsets;                 // null: one group of all rows; else [experts + 1]
  const int* order;                   // null, or the row of C for each sorted row
  void* C;
  int* partial;                       // two slots of [BT][128] per CTA
  int* counters;                      // four per CTA, one for each epilogue warp
  int64_t ldc;
  int rows, N, experts;
  int n_tiles, k_slabs;
  int BT;                             // tokens per tile
  int workers;
  int stages, stage_bytes, header, tmem_cols;
  int out_f16;
  uint32_t idesc;                     // without N
  int* status;
};

__device__ __forceinline__ float scale_of(float most) {
  return __float_as_uint(most) >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __fdiv_rn(most, 127.f);
}
__device__ __forceinline__ bool plain_scale(float s) {
  return !(fabsf(s) < 0x1p-60f || fabsf(s) > 0x1p60f) || s == 0.f;      // a NaN is as good in f32
}
// the f64 form, kept out of line: it is hardly ever reached and would crowd the instruction cache
__device__ __noinline__ float scaled(int sum, float sa, float sw, float a_max, float w_max) {
  if (plain_scale(sa) && plain_scale(sw)) return (float)sum * sa * sw;
  return (float)((double)sum * ((double)a_max / 127.0) * ((double)w_max / 127.0));
}

__device__ __forceinline__ void put(float* at, float v) { *at = v; }
__device__ __forceinline__ void put(__half* at, float v) { *at = __float2half_rn(v); }

// Up to 32 tokens of one channel: sums r scaled and stored; sa and to (row of C, negative: none) are the
// chunk's in shared memory.  `first` is the chunk's first row of C where rows are in order.
template <typename T, bool ORDERED>
__device__ __forceinline__ void store_chunk(const uint32_t (&r)[32], int count, const float* sa, const int* to, float sw, T* column,
                                            int64_t first, int64_t ldc, bool mine) {
  T* at = column + first * ldc;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 s4 = *reinterpret_cast<const float4*>(sa + i);
    const float s[4] = {s4.x, s4.y, s4.z, s4.w};
    int4 t4 = make_int4(0, 0, 0, 0);
    if (!ORDERED) t4 = *reinterpret_cast<const int4*>(to + i);
    const int t[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float v = (float)(int)r[i + j] * s[j] * sw;
      if (ORDERED) {
        if (mine && i + j < count) put(at, v);
        at += ldc;
      } else if (mine && t[j] >= 0) {
        put(column + t[j] * ldc, v);
      }
    }
  }
}

// ---------------------------------------------------------------- the schedule
// Equal contiguous runs of `total` units over `workers`: the first total % workers runs hold one more.
struct Deal {
  int64_t q, r;
  __device__ Deal(int64_t total, int workers) : q(total / workers), r(total % workers) {}
  __device__ int64_t start(int64_t w) const { return w * q + min(w, r); }
  __device__ int owner(int64_t u) const {
    const int64_t head = r * (q + 1);
    return (int)(u < head ? u / (q + 1) : r + (u - head) / q);
  }
};

struct Schedule {
  const int* row_first;     // [experts + 1] cleaned group boundaries
  const int* tile_first;    // [experts + 1] first tile of each group
  int64_t unit0, unit1;     // this worker's run
  Deal deal;                // of units, or of whole tiles
  int k_slabs;
  bool share;               // tiles may be shared
};

struct Tile {
  int expert, nt, row0, rows;
};

// Tile t (the cursor e only moves forward).
__device__ __forceinline__ Tile tile_at(const Params& p, const Schedule& s, int64_t t, int& e) {
  while (t >= s.tile_first[e + 1]) e++;
  const int first = s.row_first[e], count = s.row_first[e + 1] - first;
  const int tt = (count + p.BT - 1) / p.BT;
  const int x = (int)t - s.tile_first[e];
  const int mt = x % tt;
  return {e, x / tt, first + mt * p.BT, min(count - mt * p.BT, p.BT)};
}

// Group boundaries come from device memory: clamped and made to rise, so that nothing they hold leads
// outside the rows or covers a row twice.  One warp; tiles of a group = weight tiles x token tiles.
__device__ __forceinline__ void plan_groups(const Params& p, int w_tiles, int* row_first, int* tile_first, int lane) {
  int high = 0, tiles = 0;
  if (lane == 0) tile_first[0] = 0;
  if (!p.offsets) {
    if (lane == 0) row_first[0] = 0, row_first[1] = p.rows, tile_first[1] = w_tiles * ((p.rows + p.BT - 1) / p.BT);
    return;
  }
  for (int i0 = 0; i0 <= p.experts; i0 += 32) {
    const int i = i0 + lane;
    int v = i <= p.experts ? min(max(p.offsets[i], 0), p.rows) : 0;
    for (int d = 1; d < 32; d <<= 1) v = max(v, (int)__shfl_up_sync(0xffffffffu, v, d) * (lane >= d ? 1 : 0));
    v = max(v, high);
    int before = __shfl_up_sync(0xffffffffu, v, 1);
    if (lane == 0) before = high;                       // boundary i - 1
    high = __shfl_sync(0xffffffffu, v, 31);
    int t = (i >= 1 && i <= p.experts) ? w_tiles * ((v - before + p.BT - 1) / p.BT) : 0;
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, d);
      if (lane >= d) t += u;
    }
    t += tiles;
    if (i <= p.experts) row_first[i] = v, tile_first[i] = t;
    tiles = __shfl_sync(0xffffffffu, t, 31);
  }
}

template <bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a,
                                                                const __grid_constant__ CUtensorMap tmap_w, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);     // [kMaxStages] a stage's codes landed
  uint64_t* empty = full + kMaxStages;                     // [kMaxStages] its MMAs are done
  uint64_t* acc_full = empty + kMaxStages;                 // [2] an accumulator holds its tile
  uint64_t* acc_empty = acc_full + 2;                      // [2] its epilogue has read it
  uint64_t* drain = acc_empty + 2;                         // [1] MMAs in flight, after a give-up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* chunk_sa = reinterpret_cast<float*>(smem + 320) + ((threadIdx.x >> 5) & 3) * 32;   // [4][32] per epilogue warp
  int* chunk_to = reinterpret_cast<int*>(smem + 320 + 512) + ((threadIdx.x >> 5) & 3) * 32;
  int* row_first = reinterpret_cast<int*>(smem + kHeader);
  int* tile_first = row_first + p.experts + 1;
  uint8_t* tiles = smem + p.header;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;    // 0: the CTA that issues the pair's MMAs
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  const int w_tiles = PAIR ? (p.n_tiles + 1) / 2 : p.n_tiles;

  if (tid == 0) {
    for (int s = 0; s < kMaxStages; s++) mbar_init(smem_u32(&full[s]), PAIR ? 2 : 1), mbar_init(smem_u32(&empty[s]), 1);
    for (int b = 0; b < 2; b++) mbar_init(smem_u32(&acc_full[b]), 1), mbar_init(smem_u32(&acc_empty[b]), PAIR ? 8 : 4);
    mbar_init(smem_u32(drain), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) plan_groups(p, w_tiles, row_first, tile_first, lane);
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), (uint32_t)p.tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), (uint32_t)p.tmem_cols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();                            // both CTAs' barriers exist before either signals the other's
  tc_fence_after();
  const uint32_t own_tmem = *tmem_slot;
  // the accumulators' address is the leader's: its thread issues the MMAs for both CTAs
  const uint32_t tmem = PAIR ? ld_cluster_u32(mapa_u32(smem_u32(tmem_slot), 0)) : own_tmem;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // Deal units where that is sooner done than whole tiles, the joining of shared tiles included.
  const int64_t n_tiles_all = tile_first[p.experts], n_units = n_tiles_all * p.k_slabs;
  const int64_t whole = (n_tiles_all + p.workers - 1) / p.workers * p.k_slabs;
  const int64_t runs = min((int64_t)p.workers, max(n_units / kMinUnits, (int64_t)1));
  const bool share = (n_units + runs - 1) / runs + kSplitCost < whole;
  const int active = (int)(share ? runs : min((int64_t)p.workers, max(n_tiles_all, (int64_t)1)));
  Schedule sched{row_first, tile_first, 0, 0, Deal(share ? n_units : n_tiles_all, active), p.k_slabs, share};
  if (worker < active) {
    const int64_t grain = share ? 1 : p.k_slabs;
    sched.unit0 = sched.deal.start(worker) * grain, sched.unit1 = sched.deal.start(worker + 1) * grain;
  }
  const uint32_t ring = smem_u32(tiles);

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int s = 0, e = 0;
      uint32_t par = 0;
      int64_t issued = 0;
      bool ok = true;
      // The weights of the first ring are on their way before the codes exist (the launch that makes them
      // lets this one start when all that came before it is done, so weights and group lists are final).
      const int64_t ahead = min(sched.unit1, sched.unit0 + p.stages);
      for (int pass = 0; pass < 2; pass++) {
        if (pass) asm volatile("griddepcontrol.wait;" ::: "memory");
        s = 0, e = 0, par = 0, issued = 0;
        const int64_t stop = pass ? sched.unit1 : ahead;
        for (int64_t u = sched.unit0; u < stop && ok;) {
          const int64_t t = u / p.k_slabs;
          const Tile tile = tile_at(p, sched, t, e);
          const int64_t end = min(stop, (t + 1) * p.k_slabs);
          // a pair's second half of an odd last weight tile repeats the first; its results are not stored
          const int nt = PAIR ? min(2 * tile.nt + (int)rank, p.n_tiles - 1) : tile.nt;
          const int half = PAIR ? ((tile.rows + 31) / 32 * 32) / 2 : 0;
          const int64_t block0 = ((int64_t)tile.expert * p.n_tiles + nt) * p.k_slabs;
          for (; u < end; u++) {
            if (issued >= p.stages && !(ok = mbar_wait(smem_u32(&empty[s]), par ^ 1u, abort_flag, p.status))) break;
            const int ks = (int)(u - t * p.k_slabs);
            const uint32_t dst = ring + (uint32_t)(s * p.stage_bytes);
            // pair: both CTAs' bytes are counted on the leader's barrier
            const uint32_t bar = PAIR ? mapa_u32(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
            if (!pass || u >= ahead) {
              if (PAIR) {
                mbar_expect_tx_cluster(bar, (uint32_t)p.stage_bytes);
                tma_load_2d_pair(dst, &tmap_w, 0, (int)((block0 + ks) * 128), bar);
              } else {
                mbar_expect_tx(bar, (uint32_t)p.stage_bytes);
                bulk_load_plain(dst, p.w + (size_t)(block0 + ks) * kWTile, kWTile, bar);
              }
            }
            if (pass) {   // boxes beyond the last row are filled with zeros and count their bytes all the same
              if (PAIR) tma_load_2d_pair(dst + kWTile, &tmap_a, ks * 128, tile.row0 + (int)rank * half, bar);
              else tma_load_2d(dst + kWTile, &tmap_a, ks * 128, tile.row0, bar);
            }
            issued++;
            if (++s == p.stages) s = 0, par ^= 1u;
          }
        }
      }
      if (*abort_flag && rank == 0) {
        // copies in flight must land before the shared memory goes (the peer's count on these barriers too)
        for (int64_t i = issued > p.stages ? issued - p.stages : 0; i < issued; i++)
          for (int spin = 0; spin < 100000 && !mbar_try(smem_u32(&full[i % p.stages]), (uint32_t)(i / p.stages) & 1u); spin++) {}
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (pair: the leader's only)
    if (lane == 0 && rank == 0) {
      const uint64_t desc0 = smem_desc_sw128(ring);
      const uint32_t lo0 = (uint32_t)desc0, hi = (uint32_t)(desc0 >> 32);
      int s = 0, e = 0, seq = 0;
      uint32_t par = 0;
      bool ok = true;
      for (int64_t u = sched.unit0; u < sched.unit1 && ok; seq++) {
        const int64_t t = u / p.k_slabs;
        const Tile tile = tile_at(p, sched, t, e);
        const int64_t end = min(sched.unit1, (t + 1) * p.k_slabs);
        const int b = seq & 1;
        const int cols = PAIR ? (tile.rows + 31) / 32 * 32 : (tile.rows + 15) / 16 * 16;
        const uint32_t idesc = p.idesc | (uint32_t)(cols >> 3) << 17;
        const uint32_t acc = tmem + (uint32_t)(b * p.BT);
        if (seq >= 2 && !(ok = mbar_wait(smem_u32(&acc_empty[b]), (uint32_t)((seq >> 1) & 1) ^ 1u, abort_flag, p.status))) break;
        tc_fence_after();
        for (uint32_t first = 0; u < end; u++, first = 1) {
          if (!(ok = mbar_wait(smem_u32(&full[s]), par, abort_flag, p.status))) break;
          tc_fence_after();
          const uint32_t a_lo = lo0 + (uint32_t)((s * p.stage_bytes) >> 4);
          if (PAIR) {
            umma_i8_kblock_pair(acc, a_lo, a_lo + (kWTile >> 4), hi, idesc, first);
            umma_commit_pair(smem_u32(&empty[s]));
            umma_commit_pair(mapa_u32(smem_u32(&empty[s]), 1));
          } else {
            umma_i8_kblock(acc, a_lo, a_lo + (kWTile >> 4), hi, idesc, first);
            umma_commit(smem_u32(&empty[s]));
          }
          if (++s == p.stages) s = 0, par ^= 1u;
        }
        if (!ok) break;
        if (PAIR) {
          umma_commit_pair(smem_u32(&acc_full[b]));
          umma_commit_pair(mapa_u32(smem_u32(&acc_full[b]), 1));
        } else {
          umma_commit(smem_u32(&acc_full[b]));
        }
      }
      if (!ok) {
        if (PAIR) umma_commit_pair(smem_u32(drain));
        else umma_commit(smem_u32(drain));
        for (int spin = 0; spin < 100000 && !mbar_try(smem_u32(drain), 0); spin++) {}
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    asm volatile("griddepcontrol.wait;" ::: "memory");     // a_max and the counters are the previous launch's
    const int q = warp & 3;                                // TMEM lane quarter this warp may read
    const int ch = q * 32 + lane;                          // channel within the tile
    int e = 0, seq = 0;
    for (int64_t u = sched.unit0; u < sched.unit1; seq++) {
      const int64_t t = u / p.k_slabs;
      const Tile tile = tile_at(p, sched, t, e);
      const int64_t tile_u0 = t * p.k_slabs, tile_u1 = tile_u0 + p.k_slabs;
      const int64_t end = min(sched.unit1, tile_u1);
      const int b = seq & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[b]), (uint32_t)((seq >> 1) & 1), abort_flag, p.status))) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * p.BT);
      const int nt = PAIR ? 2 * tile.nt + (int)rank : tile.nt;
      const bool alone = u == tile_u0 && end == tile_u1;
      bool store = true;
      int w0 = 0, w1 = 0;
      if (!alone) {
        // leave the partial sums in this worker's slot; the last of the tile's workers joins them
        w0 = sched.deal.owner(tile_u0), w1 = sched.deal.owner(tile_u1 - 1);
        const int cta = PAIR ? 2 * worker + (int)rank : worker;
        int* slot = p.partial + ((size_t)cta * 2 + (u == tile_u0 ? 1 : 0)) * p.BT * 128 + ch;
        for (int c = 0; c < tile.rows; c += 32) {
          uint32_t r[32];
          tmem_ld32(acc + (uint32_t)c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i++)
            if (c + i < tile.rows) slot[(c + i) * 128] = (int)r[i];
        }
        // each warp joins its own 32 channels, so no barrier across warps is needed
        __threadfence();
        __syncwarp();
        int seen = 0;
        if (lane == 0) seen = atomicAdd(&p.counters[4 * (PAIR ? 2 * w0 + (int)rank : w0) + q], 1);
        store = __shfl_sync(0xffffffffu, seen, 0) == w1 - w0;
        __threadfence();
      }
      const int n = nt * 128 + ch;
      if (store && nt < p.n_tiles) {
        float w_max = p.w_max[((size_t)tile.expert * p.n_tiles + nt) * 128 + ch];
        const float sw = scale_of(w_max);
        if (sw != sw) w_max = sw;
        for (int c = 0; c < tile.rows; c += 32) {
          uint32_t r[32];
          tmem_ld32(acc + (uint32_t)c, r);
          float a_max = 0.f;
          int to = -1;
          if (c + lane < tile.rows) {
            const int row = tile.row0 + c + lane;
            a_max = p.a_max[row];
            to = p.order ? p.order[row] : row;
            if (to >= p.rows) to = -1;
          }
          const float sa = scale_of(a_max);
          const bool plain = __all_sync(0xffffffffu, plain_scale(sa) && plain_scale(sw));
          __syncwarp();
          chunk_sa[lane] = sa, chunk_to[lane] = to;
          __syncwarp();
          tmem_ld_wait();
          if (!alone) {
            for (int w = w0; w <= w1; w++) {
              if (w == worker) continue;
              const int cta = PAIR ? 2 * w + (int)rank : w;
              const int* slot = p.partial + ((size_t)cta * 2 + (w == w0 ? 1 : 0)) * p.BT * 128 + ch;
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (c + i < tile.rows) r[i] += (uint32_t)__ldcg(&slot[(c + i) * 128]);
            }
          }
          const bool mine = n < p.N;
          if (plain) {
            const int count = tile.rows - c;
            const int64_t first = tile.row0 + c;
            if (p.out_f16) {
              __half* column = static_cast<__half*>(p.C) + n;
              if (p.order) store_chunk<__half, false>(r, count, chunk_sa, chunk_to, sw, column, 0, p.ldc, mine);
              else store_chunk<__half, true>(r, count, chunk_sa, chunk_to, sw, column, first, p.ldc, mine);
            } else {
              float* column = static_cast<float*>(p.C) + n;
              if (p.order) store_chunk<float, false>(r, count, chunk_sa, chunk_to, sw, column, 0, p.ldc, mine);
              else store_chunk<float, true>(r, count, chunk_sa, chunk_to, sw, column, first, p.ldc, mine);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i++) {
              const int at = chunk_to[i];
              const float v = scaled((int)r[i], chunk_sa[i], sw, __shfl_sync(0xffffffffu, a_max, i), w_max);
              if (at >= 0 && mine) {
                if (p.out_f16) put(static_cast<__half*>(p.C) + at * p.ldc + n, v);
                else put(static_cast<float*>(p.C) + at * p.ldc + n, v);
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[b]), 0));
        else mbar_arrive(smem_u32(&acc_empty[b]));
      }
      u = end;
    }
  }
  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();       // the peer's MMAs read this CTA's shared memory and signal its barriers until here
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(own_tmem, (uint32_t)p.tmem_cols);
    else tmem_dealloc(own_tmem, (uint32_t)p.tmem_cols);
  }
}

// ---------------------------------------------------------------- host side
// rows of `pitch` bytes (the packed weights: whole blocks, 128-byte rows, already swizzled)
bool encode_codes(CUtensorMap* map, const void* base, int64_t pitch, int64_t rows, int box_rows, bool swizzle) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

struct Plan {
  bool pair;
  int bt, ctas;
  size_t codes, maxima, counters, partial;   // bytes of each part of the scratch
};

// Tokens per tile: a power of two that holds most groups whole (groups differ in size, so twice the mean),
// and from more than 128 on the pair form, 256 channels by 256 tokens.
bool make_plan(int64_t rows, int64_t K, int64_t experts, bool groups, Plan* pl) {
  const int64_t mean = (rows + experts - 1) / experts, want = groups ? 2 * mean : mean;
  pl->pair = mean > 128;
  pl->bt = 16;
  while (pl->bt < want && pl->bt < 128) pl->bt <<= 1;
  if (pl->pair) pl->bt = 256;
  pl->ctas = device_sm_count() & (pl->pair ? ~1 : ~0);
  pl->codes = align_up((size_t)rows * align_up((size_t)K, 128), 1024);
  pl->maxima = align_up((size_t)rows * 4, 1024);
  pl->counters = align_up((size_t)pl->ctas * 16, 1024);
  pl->partial = (size_t)pl->ctas * 2 * pl->bt * 128 * 4;
  return pl->ctas >= 2;
}

template <typename... Args>
cudaError_t launch_pdl(void (*kernel)(Args...), int cluster, int ctas, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = cluster > 1 ? 2 : 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

size_t int8_gemm_workspace_bytes(int64_t rows, int64_t K, int64_t experts, bool groups) {
  Plan pl;
  if (!make_plan(rows, K, experts, groups, &pl)) return 0;
  return pl.codes + pl.maxima + pl.counters + pl.partial;
}

cudaError_t launch_int8_gemm(const Int8Gemm& g, Workspace ws, cudaStream_t s) {
  Plan pl;
  if (!make_plan(g.rows, g.K, g.experts, g.offsets != nullptr, &pl)) return cudaErrorInvalidDevice;
  if (!ws.ptr || ws.bytes < pl.codes + pl.maxima + pl.counters + pl.partial) return cudaErrorInvalidValue;
  const int8_layout l = int8_weight_layout(g.K, g.N, g.experts);
  const int64_t kp = l.k_slabs * 128;
  uint8_t* codes = static_cast<uint8_t*>(ws.ptr);
  float* a_max = reinterpret_cast<float*>(codes + pl.codes);
  int* counters = reinterpret_cast<int*>(codes + pl.codes + pl.maxima);
  cudaError_t e = launch_int8_rows(g.dtype, g.A, g.position ? g.rows / g.fan : g.rows, g.lda, g.K, g.position, g.fan, g.rows,
                                   codes, a_max, counters, 4 * pl.ctas, s);
  if (e != cudaSuccess) return e;

  CUtensorMap map_a{}, map_w{};
  const int64_t blocks = l.experts * l.n_tiles * l.k_slabs;
  if (!encode_codes(&map_a, codes, kp, g.rows, pl.pair ? pl.bt / 2 : pl.bt, true)) return cudaErrorInvalidValue;
  if (pl.pair && (blocks * 128 > 0x7FFFFFFF || !encode_codes(&map_w, g.W, 128, blocks * 128, 128, false))) return cudaErrorInvalidValue;
  Params p{};
  p.w = static_cast<const uint8_t*>(g.W);
  p.w_max = reinterpret_cast<const float*>(p.w + l.code_bytes);
  p.a_max = a_max, p.counters = counters;
  p.partial = reinterpret_cast<int*>(codes + pl.codes + pl.maxima + pl.counters);
  p.offsets = g.offsets, p.order = g.order, p.C = g.C, p.ldc = g.ldc;
  p.rows = (int)g.rows, p.N = (int)g.N, p.experts = (int)g.experts;
  p.n_tiles = (int)l.n_tiles, p.k_slabs = (int)l.k_slabs, p.BT = pl.bt;
  p.workers = pl.pair ? pl.ctas / 2 : pl.ctas;
  p.header = (int)align_up(kHeader + (size_t)(g.experts + 1) * 8, 1024);
  p.stage_bytes = kWTile + (pl.pair ? pl.bt / 2 : pl.bt) * 128;
  p.stages = (227 * 1024 - p.header) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.tmem_cols = 2 * pl.bt < 64 ? 64 : 2 * pl.bt;           // reads go in chunks of 32 columns
  p.out_f16 = g.dtype == kDenseF16;
  // tcgen05.mma kind::i8 instruction descriptor: [4,6) D = s32 (2); [7,10) A and [10,13) B signed 8-bit (1);
  // both operands K-major; [17,23) N >> 3 (per tile); [24,29) M >> 4
  p.idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((pl.pair ? 16u : 8u) << 24);
  p.status = kernel_status_ptr();
  if (!p.status) return cudaErrorUnknown;
  static PerDeviceFlag configured;
  bool* set = configured.here();
  if (!set) return cudaErrorInvalidDevice;
  if (!*set) {
    e = cudaFuncSetAttribute(int8_gemm_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(int8_gemm_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    *set = true;
  }
  const size_t smem = p.header + (size_t)p.stages * p.stage_bytes;
  return pl.pair ? launch_pdl(int8_gemm_kernel<true>, 2, pl.ctas, smem, s, map_a, map_w, p)
                 : launch_pdl(int8_gemm_kernel<false>, 1, pl.ctas, smem, s, map_a, map_w, p);
}

}  // namespace smith
