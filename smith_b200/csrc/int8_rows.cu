// int8_rows.cu -- the 8-bit integer codes of the W8A8 products: weights packed once per channel,
// activations quantised once per token within each product.
//
// For a vector x (a weight channel or a token's activations) of finite values
//     scale = max|x| / 127,   code[k] = round-half-to-even(127 * x[k] / max|x|)   in [-127, 127]
// with the quotients taken as real numbers; a vector of zeros has scale 0 and codes 0, a vector that
// holds an infinity or a NaN has scale NaN and codes 0, so that every output it meets is NaN.  What is
// kept beside the codes is the maximum (f32, exact; NaN for a vector that is not finite), from which the
// product forms the scale.
//
// A code is evaluated in f32 and checked.  t = fma(x, f, 1.5 * 2^23) with f = f32(127 / max) rounds x * f to
// a whole number (half to even) in t's low bits; x * f is within 127 * 2^-24 < 8e-6 of the real quotient.
// Unless x * f lies closer than 2e-5 to the middle between two codes (one value in 25000) that is the
// code; otherwise the sign of 254 x - (2 low + 1) max, low being the code below, decides: each product is
// an f32 and its exact remainder (fma), the f32 parts are close and subtract exactly, and the remainders
// have few enough bits to do so too, so the sign is exact.  Vectors whose maximum is below 2^-90 or above
// 2^90 are multiplied by 2^100 or 2^-100 first, so that nothing leaves f32's range (what underflows there
// has code 0 anyway).  Conversions (f32 to integer, rint) would run at an eighth of the rate.
//
// Packed weights (built for the tensor cores' operand fetch): expert e, channel tile nt (128 channels),
// slab ks (128 k) is one contiguous block of 16 KB at ((e * NT + nt) * KS + ks) * 16384; channel r of the
// tile is 128 bytes at r * 128, and its sixteen-byte piece j stands at piece j ^ (r & 7): the 128-byte
// swizzle the MMA reads, so one plain bulk copy stages a tile.  Channels beyond N and k beyond K are
// codes 0.  The codes are followed by the channels' maxima f32 [E][NT * 128].
#include <cuda_fp16.h>

#include "int8_gemm.cuh"
#include "kernels.h"

namespace smith {
namespace {

constexpr float kTieMargin = 0.49998f;    // 0.5 - 2e-5, see above
constexpr float kMagic = 12582912.f;      // 1.5 * 2^23: adding it leaves the nearest whole number in the low bits

// How a vector's codes are made, from its maximum (finite and not 0): x * lift * factor.
struct Coder {
  float most, lift, factor;
  __device__ explicit Coder(float m) : lift(m < 0x1p-90f ? 0x1p100f : m > 0x1p90f ? 0x1p-100f : 1.f) {
    most = m * lift;
    factor = 127.f / most;
  }
};

// x (lifted) near the middle of two codes
__device__ __forceinline__ uint32_t code_near_border(float x, const Coder& c) {
  const float low = floorf(x * c.factor), odd = 2.f * low + 1.f;
  const float a = 254.f * x, b = odd * c.most;
  const float over = (a - b) + (fmaf(254.f, x, -a) - fmaf(odd, c.most, -b));
  const int l = (int)low;
  return (uint32_t)(l + (over > 0.f || (over == 0.f && (l & 1)) ? 1 : 0));
}

// The code in the low byte; off = distance of x * factor from it.
__device__ __forceinline__ uint32_t code_bits(float x, float factor, float& off) {
  const float t = fmaf(x, factor, kMagic);
  off = fabsf(fmaf(x, factor, kMagic - t));
  return __float_as_uint(t);
}

__device__ __forceinline__ uint32_t code_of(float x, const Coder& c) {
  float off;
  const uint32_t bits = code_bits(x * c.lift, c.factor, off);
  return (off > kTieMargin ? code_near_border(x * c.lift, c) : bits) & 0xFFu;
}

// bits of |x| order like |x| among non-negative f32, infinities above and NaNs above those
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
constexpr unsigned kInfBits = 0x7F800000u, kNaNBits = 0x7FC00000u;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

// ------------------------------------------------------------------------------------ weights, at load time
// Column maxima of w [E][K][N]: a block takes 256 columns and 256 rows of one expert, reads run along n.
template <typename T>
__global__ void __launch_bounds__(256) int8_column_max_kernel(const T* __restrict__ w, unsigned* __restrict__ most, int64_t K,
                                                              int64_t N, int64_t n_pad) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  const int64_t k0 = (int64_t)blockIdx.y * 256, k1 = min(k0 + 256, K);
  const T* col = w + (int64_t)blockIdx.z * K * N + n;
  unsigned m = 0;
#pragma unroll 8
  for (int64_t k = k0; k < k1; k++) m = max(m, magnitude(to_f32(col[k * N])));
  atomicMax(&most[(int64_t)blockIdx.z * n_pad + n], m);
}

// One 128 x 128 block of codes: reads along n (lanes on adjacent columns), codes of four consecutive k
// packed into a word, turned around in shared memory, stored as one contiguous 16 KB block.
template <typename T>
__global__ void __launch_bounds__(256) int8_pack_kernel(const T* __restrict__ w, uint8_t* __restrict__ codes,
                                                        const unsigned* __restrict__ most, int64_t K,
                                                        int64_t N, int64_t n_pad) {
  __shared__ __align__(16) uint32_t block[4096];
  const int64_t nt = blockIdx.x, ks = blockIdx.y, e = blockIdx.z;
  const int64_t KS = gridDim.y, NT = gridDim.x;
  const int r = threadIdx.x & 127;             // channel of the tile
  const int64_t n = nt * 128 + r;
  const unsigned bits = n < N ? most[e * n_pad + n] : 0u;
  const float m = __uint_as_float(bits);
  const bool plain = bits != 0u && bits < kInfBits;
  const Coder coder(plain ? m : 1.f);
  const T* col = w + e * K * N + n;
  for (int q = threadIdx.x >> 7; q < 32; q += 2) {   // four k each
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t k = ks * 128 + 4 * q + j;
      if (plain && k < K) word |= code_of(to_f32(col[k * N]), coder) << (8 * j);
    }
    block[r * 32 + (((q >> 2) ^ (r & 7)) << 2) + (q & 3)] = word;
  }
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(codes + ((e * NT + nt) * KS + ks) * 16384);
  const uint4* in = reinterpret_cast<const uint4*>(block);
  for (int i = threadIdx.x; i < 1024; i += 256) out[i] = in[i];
}

// ------------------------------------------------------------------------------------ activations, per product
// Sixteen bytes of a row from element k: one load, or (rows that do not start on 16 bytes, the row's end)
// value by value, zeros beyond K.  Through L2: the row may just have been written by the launch before.
template <typename T, bool WIDE>
__device__ __forceinline__ uint4 load16(const T* x, int k, int K) {
  constexpr int kVec = 16 / sizeof(T);
  if (WIDE && k + kVec <= K) return __ldcg(reinterpret_cast<const uint4*>(x + k));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (sizeof(T) == 4) {
      w[i] = k + i < K ? __ldcg(reinterpret_cast<const uint32_t*>(x) + k + i) : 0u;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(x) + k + 2 * i;
      w[i] = (k + 2 * i < K ? (uint32_t)h[0] : 0u) | (k + 2 * i + 1 < K ? (uint32_t)h[1] << 16 : 0u);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Running maximum of magnitudes as bits (halves: two in a word); infinities and NaNs are the largest.
template <typename T>
__device__ __forceinline__ void take_most(uint32_t& m, const uint4& v) {
  for (const uint32_t w : {v.x, v.y, v.z, v.w}) m = sizeof(T) == 4 ? max(m, w & 0x7FFFFFFFu) : __vmaxu2(m, w & 0x7FFF7FFFu);
}

// {lo, hi} pairs: two f32 operations in one instruction
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Codes of sixteen bytes of values.  One test for all of them decides whether any is near a border.
template <typename T>
__device__ __forceinline__ void make_codes(const uint4& raw, const Coder& coder, uint32_t (&word)[4 / sizeof(T)]) {
  constexpr int kVec = 16 / sizeof(T);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[kVec];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[(2 * i) % kVec] = f.x, x[(2 * i + 1) % kVec] = f.y;
    }
  }
  if (coder.lift != 1.f) {
#pragma unroll
    for (int j = 0; j < kVec; j++) x[j] *= coder.lift;
  }
  const uint64_t f2 = pair_of(coder.factor, coder.factor), magic2 = pair_of(kMagic, kMagic), minus2 = pair_of(-1.f, -1.f);
  uint32_t c[kVec];
  float off = 0.f;
#pragma unroll
  for (int j = 0; j < kVec; j += 2) {
    const uint64_t x2 = pair_of(x[j], x[j + 1]), t2 = fma2(x2, f2, magic2);
    float t0, t1, d0, d1;
    unpair(t2, t0, t1);
    unpair(fma2(x2, f2, fma2(t2, minus2, magic2)), d0, d1);
    c[j] = __float_as_uint(t0), c[j + 1] = __float_as_uint(t1);
    off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
  }
  if (off > kTieMargin) {
#pragma unroll
    for (int j = 0; j < kVec; j++) {
      float d;
      code_bits(x[j], coder.factor, d);
      if (d > kTieMargin) c[j] = code_near_border(x[j], coder);
    }
  }
#pragma unroll
  for (int i = 0; i < kVec / 4; i++)
    word[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
}

// One block per row of a: its maximum, then its codes (row-major, rows of kp bytes, zeros from K on) at
// the row's place, or -- with `position` -- at the `fan` places of the row in a list sorted by expert.
// A place outside [0, places) is skipped.  Each thread keeps its first kHeld vectors in registers; what a
// longer row has beyond is read again.
//
// Many rows are bound by reading them and by instructions (about six per value), few by latency: two vectors
// per thread serve both.  (4096 rows of 4096 f16: 15 to 16 us, 3.3 TB/s of reads and writes; four vectors and
// half the threads 16 to 17.  One row of 4096 f32, until the product could begin: 128 threads 5.6 us, 256
// threads 3.1, 512 threads 1.5.)  At most 32 registers a thread, so that a block of the product finds room
// beside: a quarter of an SM's register file holds three of its eleven warps, and with more registers here
// the SMs that hold one of these blocks began the product 2.5 to 5 us late.
constexpr int kNearPlaces = 32, kHeld = 2, kMostThreads = 1024;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kMostThreads, 2)
int8_rows_kernel(const T* a, int64_t lda, int K, int kp, const int* position, int fan, int places, uint8_t* codes, float* maxima,
                 int* counters, int n_counters) {
  constexpr int kVec = 16 / sizeof(T);
  // Wait first, then let the product start: what precedes this launch is finished by then, so the
  // product may read weights and group boundaries before its own wait.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t row = blockIdx.x;
  const T* x = a + row * lda;
  const int first = threadIdx.x * kVec, step = blockDim.x * kVec;
  uint4 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; i++) held[i] = first + i * step < K ? load16<T, WIDE>(x, first + i * step, K) : make_uint4(0, 0, 0, 0);
  if (blockIdx.x == 0)                       // the product's counters of shared tiles start at 0 in every call
    for (int i = threadIdx.x; i < n_counters; i += blockDim.x) counters[i] = 0;
  __shared__ unsigned warp_most[kMostThreads / 32];
  __shared__ int near_places[kNearPlaces];   // the row's places, fetched while its values are on their way
  if (threadIdx.x < kNearPlaces) near_places[threadIdx.x] = !position ? (int)row : threadIdx.x < fan ? __ldcg(&position[row * fan + threadIdx.x]) : -1;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kHeld; i++) take_most<T>(m, held[i]);
#pragma unroll 4
  for (int k = first + kHeld * step; k < K; k += step) take_most<T>(m, load16<T, WIDE>(x, k, K));
  if (sizeof(T) == 2) m = max(m & 0xFFFFu, m >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < (blockDim.x >> 5) ? warp_most[threadIdx.x & 31] : 0u);
  if (sizeof(T) == 2) m = m >= 0x7C00u ? kNaNBits : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
  const bool plain = m != 0u && m < kInfBits;
  const Coder coder(plain ? __uint_as_float(m) : 1.f);
  const int copies = position ? fan : 1;
  for (int c = threadIdx.x; c < copies; c += blockDim.x) {
    const int at = c < kNearPlaces ? near_places[c] : position[row * fan + c];
    if (at >= 0 && at < places) maxima[at] = __uint_as_float(m < kInfBits ? m : kNaNBits);
  }
  auto put_codes = [&](int k, const uint4& raw) {
    uint32_t word[kVec / 4] = {};
    if (plain) make_codes<T>(raw, coder, word);
    for (int c = 0; c < copies; c++) {
      const int at = c < kNearPlaces ? near_places[c] : position[row * fan + c];
      if (at < 0 || at >= places) continue;
      uint32_t* to = reinterpret_cast<uint32_t*>(codes + (int64_t)at * kp + k);
      if (kVec == 8) *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[kVec / 4 - 1]);
      else *to = word[0];
    }
  };
#pragma unroll
  for (int i = 0; i < kHeld; i++)
    if (first + i * step < kp) put_codes(first + i * step, held[i]);
  for (int k = first + kHeld * step; k < kp; k += step) put_codes(k, k < K ? load16<T, WIDE>(x, k, K) : make_uint4(0, 0, 0, 0));
}

}  // namespace

// ---------------------------------------------------------------------------------------------- host side
int8_layout int8_weight_layout(int64_t K, int64_t N, int64_t experts) {
  int8_layout l;
  l.n_tiles = (N + 127) / 128, l.k_slabs = (K + 127) / 128, l.experts = experts;
  l.code_bytes = (size_t)experts * l.n_tiles * l.k_slabs * 16384;
  l.bytes = l.code_bytes + (size_t)experts * l.n_tiles * 128 * 4;
  return l;
}

size_t int8_packed_bytes(int64_t K, int64_t N, int64_t experts) { return int8_weight_layout(K, N, experts).bytes; }

cudaError_t launch_int8_pack(int dtype, const void* w, void* out, int64_t K, int64_t N, int64_t experts, cudaStream_t s) {
  const int8_layout l = int8_weight_layout(K, N, experts);
  if (l.k_slabs > 65535 || experts > 65535 || l.n_tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const int64_t n_pad = l.n_tiles * 128;
  uint8_t* codes = static_cast<uint8_t*>(out);
  unsigned* most = reinterpret_cast<unsigned*>(codes + l.code_bytes);
  cudaError_t e = cudaMemsetAsync(most, 0, (size_t)experts * n_pad * 4, s);
  if (e != cudaSuccess) return e;
  const dim3 mgrid((unsigned)((N + 255) / 256), (unsigned)((K + 255) / 256), (unsigned)experts);
  const dim3 pgrid((unsigned)l.n_tiles, (unsigned)l.k_slabs, (unsigned)experts);
  if (dtype == kDenseF16) {
    int8_column_max_kernel<__half><<<mgrid, 256, 0, s>>>((const __half*)w, most, K, N, n_pad);
    int8_pack_kernel<__half><<<pgrid, 256, 0, s>>>((const __half*)w, codes, most, K, N, n_pad);
  } else {
    int8_column_max_kernel<float><<<mgrid, 256, 0, s>>>((const float*)w, most, K, N, n_pad);
    int8_pack_kernel<float><<<pgrid, 256, 0, s>>>((const float*)w, codes, most, K, N, n_pad);
  }
  count_launch(2);
  return cudaGetLastError();
}

cudaError_t launch_int8_rows(int dtype, const void* a, int64_t rows, int64_t lda, int64_t K, const int* position, int fan,
                             int64_t places, uint8_t* codes, float* maxima, int* counters, int n_counters,
                             cudaStream_t s) {
  const int64_t kp = (K + 127) / 128 * 128;
  const int es = dtype == kDenseF16 ? 2 : 4;
  const bool wide = ((reinterpret_cast<uintptr_t>(a) | (uintptr_t)(lda * es)) & 15) == 0;
  const int64_t vecs = (kp * es + 15) / 16;
  // rows fewer than SMs: at most 512 threads, which fit beside a block of the product
  const int most_threads = rows < device_sm_count() ? 512 : kMostThreads;
  int threads = 64;
  while (threads < most_threads && threads * kHeld < vecs) threads *= 2;
  using Kernel = void (*)(const void*, int64_t, int, int, const int*, int, int, uint8_t*, float*, int*, int);
  static const Kernel kernels[4] = {(Kernel)int8_rows_kernel<float, false>, (Kernel)int8_rows_kernel<float, true>,
                                    (Kernel)int8_rows_kernel<__half, false>, (Kernel)int8_rows_kernel<__half, true>};
  // The product takes nearly all of an SM's shared memory.  These blocks ask for the same split of L1 and
  // shared memory, else an SM might have to drain before it could take a block of the product.
  static PerDeviceFlag configured;
  bool* set = configured.here();
  if (!set) return cudaErrorInvalidDevice;
  if (!*set) {
    for (Kernel k : kernels) {
      const cudaError_t e = cudaFuncSetAttribute((const void*)k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
      if (e != cudaSuccess) return e;
    }
    *set = true;
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows), cfg.blockDim = dim3((unsigned)threads), cfg.stream = s;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  count_launch();
  int ikp = (int)kp, iK = (int)K, iplaces = (int)places;
  void* args[] = {&a, &lda, &iK, &ikp, &position, &fan, &iplaces, &codes, &maxima, &counters, &n_counters};
  return cudaLaunchKernelExC(&cfg, (const void*)kernels[(dtype == kDenseF16 ? 2 : 0) + (wide ? 1 : 0)], args);
}

}  // namespace smith
