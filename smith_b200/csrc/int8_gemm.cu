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
// One persistent launch.  A tile is 128 channels (a CTA pair: 256) by up to BT tokens of one group, a unit
// one slab of 128 k of a tile.  Full waves of tiles go to the workers (CTAs or pairs) whole, in blocks of
// neighbouring tiles so that what runs at one time shares its operands.  What is left after them -- often all
// there is -- is dealt in parts of tiles where that is sooner done.  A tile that two or more workers share is
// joined by the one that finishes last: the others leave their s32 partial sums in a slot of scratch and
// count themselves on a counter (zeroed by the launch that makes the codes).  Whole numbers add in any
// order, so the result does not depend on which one is last, and nobody waits.
//
// Bounds, measured on a B200 (whole call, codes included):
//   4096 x 4096 x 14336 f16   189 us = 2.5 POP/s; the product alone keeps the tensor pipe 81 % busy, at the
//                             board's power limit (SM clock 1.4 to 1.6 of 1.965 GHz); DRAM 76 MB read, the
//                             operands once
//   16 x 4096 x 14336 f32     15 us, 59 MB of weights: HBM, and about 4 us of launch, code and set-up latency
//   1 x 4096 x 4096 f32       9.5 us: latency (launch and codes 2, set-up 1.3, first weights 1.2, weights 2.6,
//                             joining 1)
// What the steps gave: loads announced without release semantics 291 -> 191 us at the largest size; MMAs
// issued by a converged warp 383 -> 183 clocks per unit; no local memory in the epilogue 264 -> 215 k clocks;
// weights and codes loaded by separate warps 480 -> 340 clocks per unit.
//
//   warp 0     weight producer: one copy of a packed 16 KB block per unit
//   warp 10    token producer: one box of codes per unit (one warp for both took 480 clocks per unit, as long
//              as the MMAs of a 256-token tile take)
//   warp 1     MMA issuer; two accumulators in tensor memory, so the next tile runs during an epilogue
//   warps 2-9  epilogue: two warps share a quarter of the lanes, each takes half of the tile's tokens
// Every mbarrier wait is time-bounded (pipeline.cuh); on a give-up the CTA waits (bounded) for its copies
// and MMAs in flight, frees its tensor memory and leaves the status word set.
#include <cuda.h>
#include <cuda_fp16.h>
#include <math.h>

#include "int8_gemm.cuh"
#include "kernels.h"
#include "pipeline.cuh"
#include "qgemv_common.cuh"
#include "tcgen05.cuh"

namespace smith {
namespace {

constexpr int kEpiWarps = 8;
constexpr int kTokenWarp = 2 + kEpiWarps;
constexpr int kThreads = (kTokenWarp + 1) * 32;
constexpr int kWTile = 16384;         // 128 channels x 128 k
constexpr int kMaxStages = 12;
constexpr int kWarpTokens = 128;      // most tokens of one epilogue warp: half of a tile
constexpr int kHeader = 512 + kEpiWarps * kWarpTokens * 8;        // barriers; the group lists follow
constexpr int kMinUnits = 2;          // fewest units per worker where runs go over tile borders
constexpr int kBlock = 16;            // token tiles side by side (4096 x 4096 x 14336: 4 -> 202 us, 8 -> 192, 16 -> 188)

struct Params {
  const uint8_t* w;
  const float* w_max;                 // [experts][n_tiles * 128]
  const float* a_max;                 // [rows]
  const int* offsets;                 // null: one group of all rows; else [experts + 1]
  const int* order;                   // null, or the row of C for each sorted row
  void* C;
  int4* partial;                      // two slots of [BT / 4][128] per CTA
  int* counters;                      // one per epilogue warp of each CTA
  float alone, join_fixed, join_each; // see Costs
  int ldc, rows, N, experts;
  int n_tiles, k_slabs;
  int w_tiles;                        // n_tiles, in pairs for the pair form
  int BT;                             // most tokens per tile
  int step;                           // tile sizes are multiples of it: 16, for a pair 32
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

// C is written once and not read here: it should not push weights and codes out of L2
__device__ __forceinline__ void put(float* at, float v) { __stcs(at, v); }
__device__ __forceinline__ void put(__half* at, float v) { __stcs(at, __float2half_rn(v)); }

// A tile's workers: w0 .. w0 + others, `worker` this one; CTAs per worker and this CTA's rank among them.
struct Sharers {
  int w0, others, worker, ctas, rank;
};

// Adds the partial sums of a tile's other workers to eight tokens.
__device__ __forceinline__ void join(const Params& p, uint32_t (&r)[8], int c, const Sharers& o, int ch) {
#pragma unroll 4
  for (int k = 0; k < o.others; k++) {
    const int w = o.w0 + k + (o.w0 + k >= o.worker ? 1 : 0);
    const int4* slot = p.partial + ((size_t)(o.ctas * w + o.rank) * 2 + (w == o.w0 ? 1 : 0)) * (p.BT * 32) + (c >> 2) * 128 + ch;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int4 v = __ldcg(&slot[i * 128]);
      r[4 * i] += (uint32_t)v.x, r[4 * i + 1] += (uint32_t)v.y, r[4 * i + 2] += (uint32_t)v.z, r[4 * i + 3] += (uint32_t)v.w;
    }
  }
}

// Tokens [c0, c1) of one channel (lane): sums read from tensor memory, the other workers' added (JOIN), scaled
// and stored.  sa and to (row of C; negative: none) are the tokens' in shared memory, from c0 on; `column` is
// the channel's element in row 0 of C (ORDERED: in the row of token c0).  Eight at a time with the next
// eight and their scales on their way.  The loop is short on purpose: the code of a small product runs once
// per launch and is paid for by its length (unrolled to 32 tokens it took 3 us), and with two warps per
// scheduler only loads ahead hide latency.
template <typename T, bool ORDERED, bool JOIN>
__device__ __forceinline__ void write_tokens(const Params& p, uint32_t acc, int c0, int c1, const float* sa, const int* to, float sw,
                                             T* column, bool mine, const Sharers& o, int ch) {
  uint64_t sw2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(sw2) : "f"(sw));
  const int ldc = p.ldc;
  uint32_t next[8];
  tmem_ld8(acc + (uint32_t)c0, next);
  ulonglong2 sa0 = *reinterpret_cast<const ulonglong2*>(sa), sa1 = *reinterpret_cast<const ulonglong2*>(sa + 4);
  T* at = column;
#pragma unroll 1
  for (int c = c0; c < c1; c += 8) {
    uint32_t r[8];
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = next[i];
    const uint64_t s[4] = {sa0.x, sa0.y, sa1.x, sa1.y};
    if (c + 8 < c1) {
      tmem_ld8(acc + (uint32_t)c + 8u, next);
      sa += 8;
      sa0 = *reinterpret_cast<const ulonglong2*>(sa), sa1 = *reinterpret_cast<const ulonglong2*>(sa + 4);
    }
    if (JOIN) join(p, r, c, o, ch);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2)      // two tokens to an instruction, each rounded as by itself
      asm("{\n.reg .b64 t;\nmov.b64 t, {%2, %3};\nmul.rn.f32x2 t, t, %4;\nmul.rn.f32x2 t, t, %5;\nmov.b64 {%0, %1}, t;\n}"
          : "=f"(v[j]), "=f"(v[j + 1])
          : "f"((float)(int)r[j]), "f"((float)(int)r[j + 1]), "l"(s[j / 2]), "l"(sw2));
    if (mine) {
      const int count = c1 - c;
      if (ORDERED && count >= 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) put(at + (int64_t)ldc * j, v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (j >= count) break;
          if (ORDERED) put(at + (int64_t)ldc * j, v[j]);
          else if (to[j] >= 0) put(column + (int64_t)ldc * to[j], v[j]);
        }
      }
    }
    if (ORDERED) at += (int64_t)ldc * 8;
    to += 8;
  }
}

// The same for a tile with a scale outside the plain range; rare, so kept out of line.
__device__ __noinline__ void write_odd(const Params& p, uint32_t acc, int c0, int c1, const float* sa, const int* to, float sw,
                                       float w_max, int row, int n, bool mine, bool joined, Sharers o, int ch) {
  for (int c = c0; c < c1; c += 8) {
    uint32_t r[8];
    tmem_ld8(acc + (uint32_t)c, r);
    tmem_ld_wait();
    if (joined) join(p, r, c, o, ch);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int i = c - c0 + j;
      if (c + j >= c1 || to[i] < 0 || !mine) continue;
      const float v = scaled((int)r[j], sa[i], sw, p.a_max[row + i], w_max);
      if (p.out_f16) put(static_cast<__half*>(p.C) + (int64_t)p.ldc * to[i] + n, v);
      else put(static_cast<float*>(p.C) + (int64_t)p.ldc * to[i] + n, v);
    }
  }
}

// ---------------------------------------------------------------- the schedule
// Equal contiguous runs of `total` units over `workers`: the first total % workers runs hold one more.
// (At most workers - 1 tiles are dealt, so there are fewer than 2^18 units.)
struct Deal {
  int q, r;
  __device__ Deal(int total, int workers) : q(total / workers), r(total - total / workers * workers) {}
  __device__ int start(int w) const { return w * q + min(w, r); }
  __device__ int owner(int u) const {
    const int head = r * (q + 1);
    return u < head ? u / (q + 1) : r + (u - head) / q;
  }
};

// A worker's work: tile i * workers + worker of each full wave, then its run of the units of what is left.
struct Schedule {
  const int* row_first;     // [experts + 1] cleaned group boundaries
  const int* tile_first;    // [experts + 1] first tile of each group
  int worker, waves;
  int shared0;              // first tile that may be shared
  int pieces;               // workers per shared tile; 0: runs go over tile borders
  Deal deal;                // units from there on
  int u, end;               // this worker's run of them
};

struct Segment {            // slabs [ks0, ks1) of a tile
  int expert, nt, row0, rows;
  int ks0, ks1;
  int unit;                 // of the tile's slab 0, counted from shared0
};

struct Walk {
  int wave = 0, e = 0;      // tiles only rise, so the group cursor only moves forward
  int u;
  __device__ explicit Walk(const Schedule& s) : u(s.u) {}
  __device__ __forceinline__ bool next(const Params& p, const Schedule& s, Segment& g) {
    int t;
    if (wave < s.waves) {
      t = wave * p.workers + s.worker;
      wave++;
      g.ks0 = 0, g.ks1 = p.k_slabs, g.unit = 0;
    } else {
      if (u >= s.end) return false;
      t = u / p.k_slabs;
      g.unit = t * p.k_slabs;
      g.ks0 = u - g.unit, g.ks1 = min(p.k_slabs, s.end - g.unit);
      u = g.unit + g.ks1;
      t += s.shared0;
    }
    while (t >= s.tile_first[e + 1]) e++;
    const int first = s.row_first[e], count = s.row_first[e + 1] - first;
    const int w_tiles = p.w_tiles;
    // blocks of up to kBlock token tiles by all weight tiles, tokens fastest: what runs at one time is
    // compact, so the codes of both sides are fetched by many workers at once
    const int tt = (count + p.BT - 1) / p.BT, x = t - s.tile_first[e];
    const int block = x / (kBlock * w_tiles), in_block = x - block * (kBlock * w_tiles);
    const int width = min(kBlock, tt - block * kBlock);
    g.nt = in_block / width;
    const int mt = block * kBlock + in_block - g.nt * width;
    // a group's tiles are of one size (300 rows: 160 and 140, not 256 and 44): a narrow tile moves the same
    // weights for less work
    const int size = ((count + tt - 1) / tt + p.step - 1) / p.step * p.step;
    g.expert = e, g.row0 = first + mt * size, g.rows = min(count - mt * size, size);
    return true;
  }
};

// Group boundaries come from device memory: clamped and made to rise, so that nothing they hold leads
// outside the rows or covers a row twice.  One warp, on row_first as fetched; tiles of a group = weight tiles
// x token tiles.
__device__ __forceinline__ void plan_groups(const Params& p, int* row_first, int* tile_first, int lane) {
  int high = 0, tiles = 0;
  if (lane == 0) tile_first[0] = 0;
  for (int i0 = 0; i0 <= p.experts; i0 += 32) {
    const int i = i0 + lane;
    int v = i <= p.experts ? row_first[i] : 0;
    for (int d = 1; d < 32; d <<= 1) v = max(v, (int)__shfl_up_sync(0xffffffffu, v, d) * (lane >= d ? 1 : 0));
    v = max(v, high);
    int before = __shfl_up_sync(0xffffffffu, v, 1);
    if (lane == 0) before = high;                       // boundary i - 1
    high = __shfl_sync(0xffffffffu, v, 31);
    int t = (i >= 1 && i <= p.experts) ? p.w_tiles * ((v - before + p.BT - 1) / p.BT) : 0;
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, d);
      if (lane >= d) t += u;
    }
    t += tiles;
    if (i <= p.experts) row_first[i] = v, tile_first[i] = t;
    tiles = __shfl_sync(0xffffffffu, t, 31);
  }
}

// The stages of a ring as one warp goes through them.  After step() the next stage's barrier is looked at
// while the warp issues what belongs to this one; wait() then often finds the answer there.
struct Ring {
  uint32_t bars;            // 8 bytes each
  int stages, s = 0;
  uint32_t par;             // phase parity that wait() expects
  bool seen = false;
  __device__ Ring(uint32_t bars, int stages, uint32_t par) : bars(bars), stages(stages), par(par) {}
  __device__ __forceinline__ bool wait(volatile int* abort_flag, int* status) {
    return seen || __all_sync(0xffffffffu, mbar_wait(bars + 8u * s, par, abort_flag, status));
  }
  __device__ __forceinline__ bool look() const {        // at the stage after this one
    const bool wrap = s + 1 == stages;
    return mbar_test(bars + (wrap ? 0u : 8u * (s + 1)), par ^ (wrap ? 1u : 0u));
  }
  __device__ __forceinline__ void step(bool looked) {
    seen = __all_sync(0xffffffffu, looked);
    if (++s == stages) s = 0, par ^= 1u;
  }
};

// Bounded time for copies in flight to land after a give-up, before the shared memory goes.
constexpr long long kLandCycles = 400000;                  // about 0.2 ms
__device__ __forceinline__ void let_copies_land() {
  const long long t0 = clock64();
  while (clock64() - t0 < kLandCycles) {}
}

template <bool PAIR>
__global__ void __maxnreg__(128)       // three warps a scheduler leave room for a block that makes codes (int8_rows.cu)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                 const __grid_constant__ Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);     // [kMaxStages] a stage's codes landed
  uint64_t* empty = full + kMaxStages;                     // [kMaxStages] its MMAs are done
  uint64_t* acc_full = empty + kMaxStages;                 // [2] an accumulator holds its tile
  uint64_t* acc_empty = acc_full + 2;                      // [2] its epilogue has read it
  uint64_t* drain = acc_empty + 2;                         // [1] MMAs in flight, after a give-up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* plan = reinterpret_cast<int*>(tmem_slot + 2);       // full waves of whole tiles; workers per tile of the rest (-1: runs)
  // per epilogue warp: scale and row of C of each of its tokens
  float* tok_sa = reinterpret_cast<float*>(smem + 512) + ((threadIdx.x >> 5) & 7) * kWarpTokens;
  int* tok_to = reinterpret_cast<int*>(smem + 512 + kEpiWarps * kWarpTokens * 4) + ((threadIdx.x >> 5) & 7) * kWarpTokens;
  int* row_first = reinterpret_cast<int*>(smem + kHeader);
  int* tile_first = row_first + p.experts + 1;
  uint8_t* tiles = smem + p.header;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;    // 0: the CTA that issues the pair's MMAs
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x;

  if (warp == 2) {                       // a lane per barrier
    if (lane < kMaxStages) mbar_init(smem_u32(&full[lane]), PAIR ? 2 : 1), mbar_init(smem_u32(&empty[lane]), 1);
    else if (lane < kMaxStages + 2) mbar_init(smem_u32(&acc_full[lane - kMaxStages]), 1);
    else if (lane < kMaxStages + 4) mbar_init(smem_u32(&acc_empty[lane - kMaxStages - 2]), (PAIR ? 2 : 1) * kEpiWarps);
    else if (lane == kMaxStages + 4) mbar_init(smem_u32(drain), 1), *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), (uint32_t)p.tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), (uint32_t)p.tmem_cols);
      tmem_relinquish();
    }
  }
  if (warp == 0) {
    if (p.offsets) {
#pragma unroll 4
      for (int i = lane; i <= p.experts; i += 32) row_first[i] = min(max(__ldcg(&p.offsets[i]), 0), p.rows);
      __syncwarp();
      plan_groups(p, row_first, tile_first, lane);
    } else if (lane == 0) {
      row_first[0] = 0, row_first[1] = p.rows;
      tile_first[0] = 0, tile_first[1] = p.w_tiles * ((p.rows + p.BT - 1) / p.BT);
    }
    __syncwarp();
    // What is left after the full waves: whole tiles (lane 0), l + 1 workers per tile (lane l), or runs of
    // units over all workers (lane 31), whichever is done first.  A worker alone moves its units faster
    // than its share of the memory's rate (p.alone), so few workers can be enough; joining costs
    // p.join_fixed units per shared tile of a worker and p.join_each per other worker of the tile.
    const int n_all = tile_first[p.experts], waves = n_all / p.workers, left = n_all - waves * p.workers;
    const int all = left * p.k_slabs;
    int each = (p.k_slabs + lane) / (lane + 1);
    float joins = lane == 0 ? 0.f : p.join_fixed + p.join_each * (float)lane;
    bool can = left * (lane + 1) <= p.workers && lane < p.k_slabs;
    if (lane == 31) {
      each = (all + p.workers - 1) / p.workers;
      can = each >= kMinUnits;
      joins = 2.f * p.join_fixed + p.join_each * (float)(1 + p.k_slabs / max(each, 1));
    }
    const float cost = can ? fmaxf((float)all / (float)p.workers, p.alone * (float)each) + joins : 1e30f;
    const unsigned bits = __float_as_uint(cost), least = __reduce_min_sync(0xffffffffu, bits);
    const int best = __ffs(__ballot_sync(0xffffffffu, bits == least)) - 1;
    if (lane == best) plan[0] = waves, plan[1] = lane == 31 ? -1 : lane + 1;
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();                            // both CTAs' barriers exist before either signals the other's
  tc_fence_after();
  const uint32_t own_tmem = *tmem_slot;
  // the accumulators' address is the leader's: its thread issues the MMAs for both CTAs
  const uint32_t tmem = PAIR ? ld_cluster_u32(mapa_u32(smem_u32(tmem_slot), 0)) : own_tmem;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int waves = plan[0], pieces = plan[1], n_all = tile_first[p.experts], shared0 = waves * p.workers;
  const int left = n_all - shared0;
  Schedule sched{row_first, tile_first, worker, waves, shared0, max(pieces, 0), Deal(left * p.k_slabs, p.workers), 0, 0};
  if (pieces < 0) {                                             // runs over all units
    sched.u = sched.deal.start(worker), sched.end = sched.deal.start(worker + 1);
  } else if (pieces > 1) {
    const int t = worker / pieces;
    const Deal slabs(p.k_slabs, pieces);
    if (t < left) sched.u = t * p.k_slabs + slabs.start(worker - t * pieces), sched.end = t * p.k_slabs + slabs.start(worker - t * pieces + 1);
  } else {
    sched.waves += shared0 + worker < n_all;                    // whole tiles: one more for the first workers
  }
  const uint32_t ring = smem_u32(tiles);

  if (warp == 0) {
    // ------------------------------------------------------------ weight producer (the whole warp; one lane issues)
    // Does not wait for the launch that makes the codes: that one lets this one start when all that came
    // before it is done, so weights and group lists are final.  The first ring is on its way by then.
    const uint32_t bytes = (uint32_t)p.stage_bytes;
    // pair: both CTAs' bytes are counted on the leader's barriers
    const uint32_t bar0 = PAIR ? mapa_u32(smem_u32(full), 0) : smem_u32(full);
    Ring r(smem_u32(empty), p.stages, 1u);                 // a fresh barrier is past phase "1": nothing to wait for
    bool ok = true;
    Walk walk(sched);
    Segment g;
    while (ok && walk.next(p, sched, g)) {
      // a pair's second half of an odd last weight tile repeats the first; its results are not stored
      const int nt = PAIR ? min(2 * g.nt + (int)rank, p.n_tiles - 1) : g.nt;
      const int64_t block0 = ((int64_t)g.expert * p.n_tiles + nt) * p.k_slabs;
      for (int ks = g.ks0; ks < g.ks1; ks++) {
        if (!(ok = r.wait(abort_flag, p.status))) break;
        const bool looked = r.look();
        const uint32_t dst = ring + (uint32_t)r.s * bytes, bar = bar0 + 8u * r.s;
        if (PAIR) {
          mbar_expect_tx_cluster_elected(bar, bytes);
          tma_load_2d_pair_elected(dst, &tmap_w, 0, (int)((block0 + ks) * (kWTile / 1024)), bar);
        } else {
          mbar_expect_tx_elected(bar, bytes);
          bulk_load_elected(dst, p.w + (size_t)(block0 + ks) * kWTile, kWTile, bar);
        }
        r.step(looked);
      }
    }
    if (!ok) let_copies_land();
  } else if (warp == kTokenWarp) {
    // ------------------------------------------------------------ token producer
    asm volatile("griddepcontrol.wait;" ::: "memory");     // the codes are the previous launch's
    const uint32_t bytes = (uint32_t)p.stage_bytes;
    const uint32_t bar0 = PAIR ? mapa_u32(smem_u32(full), 0) : smem_u32(full);
    Ring r(smem_u32(empty), p.stages, 1u);
    bool ok = true;
    Walk walk(sched);
    Segment g;
    while (ok && walk.next(p, sched, g)) {
      const int row = g.row0 + (PAIR ? (int)rank * (((g.rows + 31) / 32 * 32) / 2) : 0);
      for (int ks = g.ks0; ks < g.ks1; ks++) {
        if (!(ok = r.wait(abort_flag, p.status))) break;
        const bool looked = r.look();
        const uint32_t dst = ring + (uint32_t)r.s * bytes + kWTile, bar = bar0 + 8u * r.s;
        // a box beyond the last row is filled with zeros and counts its bytes all the same
        if (PAIR) tma_load_2d_pair_elected(dst, &tmap_a, ks * 128, row, bar);
        else tma_load_2d_elected(dst, &tmap_a, ks * 128, row, bar);
        r.step(looked);
      }
    }
    if (!ok) let_copies_land();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (pair: the leader's only)
    if (rank == 0) {
      const uint64_t desc0 = smem_desc_sw128(ring);
      const uint32_t lo0 = (uint32_t)desc0, hi = (uint32_t)(desc0 >> 32), step = (uint32_t)p.stage_bytes >> 4;
      int seq = 0;
      bool ok = true;
      Ring r(smem_u32(full), p.stages, 0u);
      Walk walk(sched);
      Segment g;
      for (; ok && walk.next(p, sched, g); seq++) {
        const int b = seq & 1;
        const int cols = PAIR ? (g.rows + 31) / 32 * 32 : (g.rows + 15) / 16 * 16;
        const uint32_t idesc = p.idesc | (uint32_t)(cols >> 3) << 17;
        const uint32_t acc = tmem + (uint32_t)(b * p.BT);
        if (seq >= 2) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_empty[b]), (uint32_t)((seq >> 1) & 1) ^ 1u, abort_flag, p.status));
        if (!ok) break;
        tc_fence_after();
        uint32_t first = 0;
        for (int ks = g.ks0; ks < g.ks1; ks++, first = 1) {
          if (!(ok = r.wait(abort_flag, p.status))) break;
          tc_fence_after();
          const bool looked = r.look();
          const uint32_t a_lo = lo0 + (uint32_t)r.s * step, done = smem_u32(empty) + 8u * r.s;
          if (PAIR) {
            umma_i8_kblock_pair(acc, a_lo, a_lo + (kWTile >> 4), hi, idesc, first);
            umma_commit_both_elected(done);
          } else {
            umma_i8_kblock(acc, a_lo, a_lo + (kWTile >> 4), hi, idesc, first);
            umma_commit_elected(done);
          }
          r.step(looked);
        }
        if (!ok) break;
        if (PAIR) umma_commit_both_elected(smem_u32(&acc_full[b]));
        else umma_commit_elected(smem_u32(&acc_full[b]));
      }
      if (!ok) {
        if (PAIR) umma_commit_both_elected(smem_u32(drain));
        else umma_commit_elected(smem_u32(drain));
        const long long t0 = clock64();
        while (!mbar_try(smem_u32(drain), 0) && clock64() - t0 < kLandCycles) {}
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    asm volatile("griddepcontrol.wait;" ::: "memory");     // a_max and the counters are the previous launch's
    const int q = warp & 3;                                // TMEM lane quarter this warp may read
    const int ch = q * 32 + lane;                          // channel within the tile
    const bool second = warp >= 2 + 4;                     // of the two warps of this quarter
    int seq = 0;
    Walk walk(sched);
    Segment tile;
    for (; walk.next(p, sched, tile); seq++) {
      const int b = seq & 1;
      const int nt = PAIR ? 2 * tile.nt + (int)rank : tile.nt;
      const int n = nt * 128 + ch;
      const bool alone = tile.ks1 - tile.ks0 == p.k_slabs;
      const bool mine = nt < p.n_tiles && n < p.N;
      const int half = ((tile.rows + 1) / 2 + 7) & ~7;
      const int c0 = second ? half : 0, c1 = second ? tile.rows : min(half, tile.rows);
      // what the results need is fetched while the tile is still being multiplied
      float w_max = mine ? p.w_max[((size_t)tile.expert * p.n_tiles + nt) * 128 + ch] : 0.f;
      const float sw = scale_of(w_max);
      if (sw != sw) w_max = sw;
      bool plain = plain_scale(sw);
      __syncwarp();
      for (int i = lane; c0 + i < c1; i += 32) {
        const int row = tile.row0 + c0 + i;
        const float sa = scale_of(__ldcg(&p.a_max[row]));
        const int to = p.order ? __ldcg(&p.order[row]) : row;
        tok_sa[i] = sa, tok_to[i] = to < p.rows ? to : -1;
        plain = plain && plain_scale(sa);
      }
      plain = __all_sync(0xffffffffu, plain);
      __syncwarp();
      int w0 = 0, others = 0, seen = 0;
      int* counter = nullptr;
      if (!alone) {
        if (sched.pieces) w0 = tile.unit / p.k_slabs * sched.pieces, others = sched.pieces - 1;
        else w0 = sched.deal.owner(tile.unit), others = sched.deal.owner(tile.unit + p.k_slabs - 1) - w0;
        counter = &p.counters[kEpiWarps * (PAIR ? 2 * w0 + (int)rank : w0) + warp - 2];
        if (lane == 0) asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
        seen = __shfl_sync(0xffffffffu, seen, 0);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[b]), (uint32_t)((seq >> 1) & 1), abort_flag, p.status))) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * p.BT);
      bool store = c0 < c1;
      if (!alone && c0 < c1) {
        // Leave the partial sums in this worker's slot; the last of the tile's workers joins them.  Each warp
        // joins its own channels and tokens, so no barrier across warps is needed.  A worker that finds all
        // others done is the last and need not write its own sums.
        if (seen != others) {
          const int cta = PAIR ? 2 * worker + (int)rank : worker;
          int4* slot = p.partial + ((size_t)cta * 2 + (tile.ks0 == 0 ? 1 : 0)) * (p.BT * 32) + ch;
#pragma unroll 1
          for (int c = c0; c < c1; c += 8) {
            uint32_t r[8];
            tmem_ld8(acc + (uint32_t)c, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; i += 4)
              slot[((c + i) >> 2) * 128] = make_int4((int)r[i], (int)r[i + 1], (int)r[i + 2], (int)r[i + 3]);
          }
          __threadfence();
          __syncwarp();
          if (lane == 0) seen = atomicAdd(counter, 1);
          store = __shfl_sync(0xffffffffu, seen, 0) == others;
        }
        if (store) __threadfence();
      }
      if (store && nt < p.n_tiles) {
        const Sharers o{w0, others, worker, PAIR ? 2 : 1, (int)rank};
        const bool ordered = !p.order;
        const int64_t first = (ordered ? (int64_t)p.ldc * (tile.row0 + c0) : 0) + n;
        float* C32 = static_cast<float*>(p.C) + first;
        __half* C16 = static_cast<__half*>(p.C) + first;
        if (!plain) write_odd(p, acc, c0, c1, tok_sa, tok_to, sw, w_max, tile.row0 + c0, n, mine, !alone, o, ch);
        else if (alone && ordered && p.out_f16) write_tokens<__half, true, false>(p, acc, c0, c1, tok_sa, tok_to, sw, C16, mine, o, ch);
        else if (alone && ordered) write_tokens<float, true, false>(p, acc, c0, c1, tok_sa, tok_to, sw, C32, mine, o, ch);
        else if (ordered && p.out_f16) write_tokens<__half, true, true>(p, acc, c0, c1, tok_sa, tok_to, sw, C16, mine, o, ch);
        else if (ordered) write_tokens<float, true, true>(p, acc, c0, c1, tok_sa, tok_to, sw, C32, mine, o, ch);
        else if (alone && p.out_f16) write_tokens<__half, false, false>(p, acc, c0, c1, tok_sa, tok_to, sw, C16, mine, o, ch);
        else if (alone) write_tokens<float, false, false>(p, acc, c0, c1, tok_sa, tok_to, sw, C32, mine, o, ch);
        else if (p.out_f16) write_tokens<__half, false, true>(p, acc, c0, c1, tok_sa, tok_to, sw, C16, mine, o, ch);
        else write_tokens<float, false, true>(p, acc, c0, c1, tok_sa, tok_to, sw, C32, mine, o, ch);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[b]), 0));
        else mbar_arrive(smem_u32(&acc_empty[b]));
      }
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
bool encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t inner, int64_t rows, int64_t pitch, int box_inner,
                int box_rows, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// token codes [rows][kp], boxes of 128 k in the 128-byte swizzle
bool encode_codes(CUtensorMap* map, const void* base, int64_t kp, int64_t rows, int box_rows) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, kp, rows, kp, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}
// packed weights as lines of 1 KB, sixteen to a block, copied as they are
constexpr int kBlockLines = kWTile / 1024;
bool encode_blocks(CUtensorMap* map, const void* base, int64_t blocks) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_INT32, base, 256, blocks * kBlockLines, 1024, 256, kBlockLines, CU_TENSOR_MAP_SWIZZLE_NONE);
}

size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

// In units of the main loop (0.28 us for a pair at 256 tokens, bound by the tensor cores; 0.37 us for one
// CTA of 148 that stream weights): the time of a unit when few workers are active, what a worker pays once
// for a shared tile (writing, the counter, the stores), and for the sums of each other worker.
struct Costs {
  double alone, join_fixed, join_each;
  Costs(bool pair, int bt) : alone(pair ? 1.0 : 0.65), join_fixed(pair ? 11.0 : 4.0 + 3.0 * bt / 128), join_each(pair ? 7.0 : 0.5 + 2.0 * bt / 128) {}
};

struct Plan {
  bool pair;
  int bt, ctas;
  size_t codes, maxima, counters, partial;   // bytes of each part of the scratch
};

// Tokens per tile.  Few tokens: a power of two that holds most groups whole (groups differ in size, so twice
// the mean).  More than 128: the pair form, 256 channels by up to 256 tokens; for one matrix the width that
// leaves the least idle in the last wave.  A unit takes 2 clocks per token and a part that does not shrink
// with the width: at full rate the board is at its power limit, and the weights' way through L2 costs the
// same for a narrow tile (measured at 4096 x 4096 x 14336: 256 wide 229 us, the narrower tile that an equal
// price per token would choose 290 us).
bool make_plan(int64_t rows, int64_t N, int64_t K, int64_t experts, bool groups, Plan* pl) {
  const int64_t mean = (rows + experts - 1) / experts, want = groups ? 2 * mean : mean;
  pl->ctas = device_sm_count();
  pl->pair = mean > 128;
  pl->bt = 16;
  while (pl->bt < want && pl->bt < 128) pl->bt <<= 1;
  if (pl->pair) {
    pl->ctas &= ~1;
    pl->bt = 256;
    double least = 0;
    const int64_t slabs = (K + 127) / 128, w_tiles = (N + 255) / 256, workers = pl->ctas / 2;
    // (of many waves the last is a small part: the widest tile then)
    for (int64_t tt = (rows + 255) / 256; !groups && tt <= (rows + 127) / 128 && tt * w_tiles < 16 * workers; tt++) {
      const int bt = (int)(((rows + tt - 1) / tt + 31) / 32 * 32);
      const int64_t tiles = w_tiles * tt, left = tiles % workers;
      const Costs c(true, bt);
      double tail = left ? (double)slabs : 0;
      for (int64_t pieces = 2; left && left * pieces <= workers && pieces <= slabs; pieces++) {
        const double t = (double)((slabs + pieces - 1) / pieces) + c.join_fixed + c.join_each * (pieces - 1);
        if (t < tail) tail = t;
      }
      const double run = ceil((double)(left * slabs) / workers);
      if (left && run >= kMinUnits && run + 2 * c.join_fixed + c.join_each * (1 + slabs / run) < tail)
        tail = run + 2 * c.join_fixed + c.join_each * (1 + slabs / run);
      const double cost = ((double)(tiles / workers * slabs) + tail) * (bt * 2 + 130);
      if (least == 0 || cost < least) least = cost, pl->bt = bt;
    }
  }
  pl->codes = align_up((size_t)rows * align_up((size_t)K, 128), 1024);
  pl->maxima = align_up((size_t)rows * 4, 1024);
  pl->counters = align_up((size_t)pl->ctas * kEpiWarps * 4, 1024);
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

size_t int8_gemm_workspace_bytes(int64_t rows, int64_t N, int64_t K, int64_t experts, bool groups) {
  Plan pl;
  if (!make_plan(rows, N, K, experts, groups, &pl)) return 0;
  return pl.codes + pl.maxima + pl.counters + pl.partial;
}

cudaError_t launch_int8_gemm(const Int8Gemm& g, Workspace ws, cudaStream_t s) {
  Plan pl;
  if (!make_plan(g.rows, g.N, g.K, g.experts, g.offsets != nullptr, &pl)) return cudaErrorInvalidDevice;
  if (!ws.ptr || ws.bytes < pl.codes + pl.maxima + pl.counters + pl.partial) return cudaErrorInvalidValue;
  const int8_layout l = int8_weight_layout(g.K, g.N, g.experts);
  const int64_t kp = l.k_slabs * 128;
  uint8_t* codes = static_cast<uint8_t*>(ws.ptr);
  float* a_max = reinterpret_cast<float*>(codes + pl.codes);
  int* counters = reinterpret_cast<int*>(codes + pl.codes + pl.maxima);
  cudaError_t e = launch_int8_rows(g.dtype, g.A, g.position ? g.rows / g.fan : g.rows, g.lda, g.K, g.position, g.fan, g.rows,
                                   codes, a_max, counters, kEpiWarps * pl.ctas, s);
  if (e != cudaSuccess) return e;

  CUtensorMap map_a{}, map_w{};
  const int64_t blocks = l.experts * l.n_tiles * l.k_slabs;
  const int box = pl.pair ? pl.bt / 2 : pl.bt;              // token codes a CTA stages per unit
  if (!encode_codes(&map_a, codes, kp, g.rows, box)) return cudaErrorInvalidValue;
  if (pl.pair && (blocks * kBlockLines > 0x7FFFFFFF || !encode_blocks(&map_w, g.W, blocks))) return cudaErrorInvalidValue;
  Params p{};
  p.w = static_cast<const uint8_t*>(g.W);
  p.w_max = reinterpret_cast<const float*>(p.w + l.code_bytes);
  p.a_max = a_max, p.counters = counters;
  const Costs costs(pl.pair, pl.bt);
  p.alone = (float)costs.alone, p.join_fixed = (float)costs.join_fixed, p.join_each = (float)costs.join_each;
  p.partial = reinterpret_cast<int4*>(codes + pl.codes + pl.maxima + pl.counters);
  p.offsets = g.offsets, p.order = g.order, p.C = g.C, p.ldc = (int)g.ldc;
  p.rows = (int)g.rows, p.N = (int)g.N, p.experts = (int)g.experts;
  p.n_tiles = (int)l.n_tiles, p.k_slabs = (int)l.k_slabs, p.BT = pl.bt;
  p.w_tiles = pl.pair ? (p.n_tiles + 1) / 2 : p.n_tiles;
  p.workers = pl.pair ? pl.ctas / 2 : pl.ctas;
  p.header = (int)align_up(kHeader + (size_t)(g.experts + 1) * 8, 1024);
  p.step = pl.pair ? 32 : 16;
  p.stage_bytes = kWTile + box * 128;
  p.stages = (227 * 1024 - p.header) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.tmem_cols = 32;                                        // a power of two, 32 at least
  while (p.tmem_cols < 2 * pl.bt) p.tmem_cols <<= 1;
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
