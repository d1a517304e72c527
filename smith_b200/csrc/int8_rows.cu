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
// A code is evaluated in f32 and checked: q = x * (127 / max) carries two roundings, |q| <= 127, so it is
// within 127 * (2^-23 + 2^-48) < 1.6e-5 of the real quotient.  Unless q lies closer than 2e-5 to the
// middle between two codes (one value in 25000) the nearest integer to q is the code; otherwise, and for
// vectors so small that 127 / max leaves f32, the quotient is formed in f64: 127 * x is exact there, and
// a quotient of a 31-bit and a 24-bit number that is no half-integer differs from every half-integer by
// far more than an f64 rounding, so the result is the definition's in every case.
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
constexpr float kSmallMax = 1e-30f;       // below this 127 / max would leave f32's range soon: all in f64

// 127 / max, or 0 where no f32 value serves (the f64 lane takes over; `max` must not be 0)
__device__ __forceinline__ float code_factor(float most) { return most >= kSmallMax ? 127.f / most : 0.f; }

// out of line: reached for one value in 25000, and it would crowd the instruction cache
__device__ __noinline__ int code_f64(float x, float most) { return (int)rint(__dmul_rn((double)x, 127.0) / (double)most); }

__device__ __forceinline__ int code_of(float x, float most, float factor) {
  const float q = x * factor;
  const float r = rintf(q);
  if (fabsf(q - r) > kTieMargin || factor == 0.f) return code_f64(x, most);
  return (int)r;
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
  const float factor = plain ? code_factor(m) : 0.f;
  const T* col = w + e * K * N + n;
  for (int q = threadIdx.x >> 7; q < 32; q += 2) {   // four k each
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t k = ks * 128 + 4 * q + j;
      if (plain && k < K) word |= (uint32_t)(code_of(to_f32(col[k * N]), m, factor) & 0xFF) << (8 * j);
    }
    block[r * 32 + (((q >> 2) ^ (r & 7)) << 2) + (q & 3)] = word;
  }
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(codes + ((e * NT + nt) * KS + ks) * 16384);
  const uint4* in = reinterpret_cast<const uint4*>(block);
  for (int i = threadIdx.x; i < 1024; i += 256) out[i] = in[i];
}

// ------------------------------------------------------------------------------------ activations, per product
// kVec consecutive values of a row as f32: one 16-byte load, or (rows that do not start on 16 bytes, the
// row's end) value by value, zeros beyond K.
template <typename T>
struct RowVec;
template <>
struct RowVec<float> {
  static constexpr int kVec = 4;
  __device__ static void load16(const float* x, float (&v)[4]) {
    const float4 t = *reinterpret_cast<const float4*>(x);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  }
};
template <>
struct RowVec<__half> {
  static constexpr int kVec = 8;
  __device__ static void load16(const __half* x, float (&v)[8]) {
    const uint4 t = *reinterpret_cast<const uint4*>(x);
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load_row(const T* x, int64_t k, int64_t K, float (&v)[RowVec<T>::kVec]) {
  constexpr int kVec = RowVec<T>::kVec;
  if (WIDE && k + kVec <= K) {
    RowVec<T>::load16(x + k, v);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; j++) v[j] = k + j < K ? to_f32(x[k + j]) : 0.f;
  }
}

// Codes of kVec values as bytes.  One test for all of them decides whether any is near a border.
template <int kVec>
__device__ __forceinline__ void make_codes(const float (&v)[kVec], float most, float factor, uint32_t (&word)[kVec / 4]) {
  int c[kVec];
  float off = 0.f;
#pragma unroll
  for (int j = 0; j < kVec; j++) {
    const float q = v[j] * factor, r = rintf(q);
    off = fmaxf(off, fabsf(q - r));
    c[j] = (int)r;
  }
  if (off > kTieMargin || factor == 0.f) {
#pragma unroll
    for (int j = 0; j < kVec; j++) c[j] = code_f64(v[j], most);
  }
#pragma unroll
  for (int i = 0; i < kVec / 4; i++)
    word[i] = (uint32_t)(c[4 * i] & 0xFF) | (uint32_t)(c[4 * i + 1] & 0xFF) << 8 | (uint32_t)(c[4 * i + 2] & 0xFF) << 16 |
              (uint32_t)(c[4 * i + 3] & 0xFF) << 24;
}

// One block per row of a: its maximum, then its codes (row-major, rows of kp bytes, zeros from K on) at
// the row's place, or -- with `position` -- at the `fan` places of the row in a list sorted by expert.
// A place outside [0, places) is skipped.  The second reading of the row finds it in L1 or L2.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(1024) int8_rows_kernel(const T* a, int64_t lda, int64_t K, int64_t kp, const int* position, int fan,
                                                         int64_t places, uint8_t* codes, float* maxima, int* counters,
                                                         int n_counters) {
  constexpr int kVec = RowVec<T>::kVec;
  // Wait first, then let the product start: what precedes this launch is finished by then, so the
  // product may read weights and group boundaries before its own wait.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x == 0)                       // the product's counters of shared tiles start at 0 in every call
    for (int i = threadIdx.x; i < n_counters; i += blockDim.x) counters[i] = 0;
  __shared__ unsigned warp_most[32];
  const int64_t row = blockIdx.x;
  const T* x = a + row * lda;
  const int64_t step = (int64_t)blockDim.x * kVec;
  unsigned m = 0;
#pragma unroll 4
  for (int64_t k = (int64_t)threadIdx.x * kVec; k < K; k += step) {
    float v[kVec];
    load_row<T, WIDE>(x, k, K, v);
#pragma unroll
    for (int j = 0; j < kVec; j++) m = max(m, magnitude(v[j]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < (blockDim.x >> 5) ? warp_most[threadIdx.x & 31] : 0u);
  const bool plain = m != 0u && m < kInfBits;
  const float most = __uint_as_float(m), factor = plain ? code_factor(most) : 0.f;
  const int copies = position ? fan : 1;
  for (int c = threadIdx.x; c < copies; c += blockDim.x) {
    const int64_t at = position ? (int64_t)position[row * fan + c] : row;
    if (at >= 0 && at < places) maxima[at] = __uint_as_float(m < kInfBits ? m : kNaNBits);
  }
#pragma unroll 2
  for (int64_t k = (int64_t)threadIdx.x * kVec; k < kp; k += step) {
    uint32_t word[kVec / 4] = {};
    if (plain) {
      float v[kVec];
      load_row<T, WIDE>(x, k, K, v);
      make_codes<kVec>(v, most, factor, word);
    }
    for (int c = 0; c < copies; c++) {
      const int64_t at = position ? (int64_t)position[row * fan + c] : row;
      if (at < 0 || at >= places) continue;
      uint32_t* to = reinterpret_cast<uint32_t*>(codes + at * kp + k);
      if (kVec == 8) *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[kVec / 4 - 1]);
      else *to = word[0];
    }
  }
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
  // threads: four 16-byte loads each, two where there are fewer rows than SMs and latency counts
  const int64_t vecs = (kp * es + 15) / 16, each = rows < device_sm_count() ? 2 : 4;
  int threads = 64;
  while (threads < 1024 && threads * each < vecs) threads *= 2;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows), cfg.blockDim = dim3((unsigned)threads), cfg.stream = s;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  count_launch();
  if (dtype == kDenseF16)
    return cudaLaunchKernelEx(&cfg, wide ? int8_rows_kernel<__half, true> : int8_rows_kernel<__half, false>, (const __half*)a, lda, K,
                              kp, position, fan, places, codes, maxima, counters, n_counters);
  return cudaLaunchKernelEx(&cfg, wide ? int8_rows_kernel<float, true> : int8_rows_kernel<float, false>, (const float*)a, lda, K, kp,
                            position, fan, places, codes, maxima, counters, n_counters);
}

}  // namespace smith
