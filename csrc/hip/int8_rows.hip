// Rows to 8-bit integers with one scale per row (gfx950): plain rows, the root-mean-square norm with the
// residual's addition, and the gated activation of an MLP; and the way back.
//
//   p      the row in fp32:  x  |  round_T(x + r) * w  |  g / (1 + exp(-g)) * u
//   m      max |p|
//   q_k    the integer nearest to 127 p_k / m, ties to even
//   s      m f / 127 with f = 1, or 1 / sqrt(mean(h^2) + eps) for the norm of h = round_T(x + r)
//
// The norm's factor f is the same for the whole row, so it cancels in q: the integers come from h w alone and f only
// enters the scale.  One pass over the row therefore suffices: it is loaded once into registers, the maximum and the
// sum of squares are reduced together, and the integers leave from the registers.  The kernels are bound by memory.
//
// q is decided exactly.  t = p * (127 / m) in fp32 carries two roundings of 2^-24 on a value up to 127, at most
// 1.6e-5; where t lies within 4e-5 of a border between two integers (one value in about 10^4) the quotient is taken
// in 64 bits, where 127 p is exact and no quotient of two fp32 numbers that is not a border rounds to one.
//
// A row with m = 0 gives q = 0 and s = 0.  A row in which any p is not finite gives q = 0 and s = NaN: integers have
// no NaN, so the scale carries it and whatever is computed from the row is NaN.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace {

using half8 = __attribute__((ext_vector_type(8))) _Float16;
using ushort8 = __attribute__((ext_vector_type(8))) unsigned short;
using float4v = __attribute__((ext_vector_type(4))) float;

constexpr int kVec = 8;  // values per chunk: one 16-byte load of a 16-bit type, one 8-byte store of integers

enum Mode : int { kPlain = 0, kNorm = 1, kNormResidual = 2, kGate = 3 };

struct Bf16 {
  unsigned short bits;
};

// ---- chunks of eight values; addresses need no alignment beyond the element's own --------------------------------

__device__ __forceinline__ void Unpack(const float* p, float (&v)[kVec]) {
  __builtin_memcpy(v, p, sizeof(v));
}
__device__ __forceinline__ void Unpack(const _Float16* p, float (&v)[kVec]) {
  half8 h;
  __builtin_memcpy(&h, p, sizeof(h));
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = static_cast<float>(h[i]);
}
__device__ __forceinline__ void Unpack(const Bf16* p, float (&v)[kVec]) {
  ushort8 h;
  __builtin_memcpy(&h, p, sizeof(h));
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = __uint_as_float(static_cast<unsigned>(h[i]) << 16);
}

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(_Float16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float ToFloat(Bf16 v) { return __uint_as_float(static_cast<unsigned>(v.bits) << 16); }

template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 FromFloat<_Float16>(float v) { return static_cast<_Float16>(v); }
template <> __device__ __forceinline__ Bf16 FromFloat<Bf16>(float v) {
  return Bf16{__builtin_bit_cast(unsigned short, static_cast<__bf16>(v))};  // nearest, ties to even, NaN kept
}

template <typename T>
__device__ __forceinline__ void LoadChunk(const T* row, int first, int width, float (&v)[kVec]) {
  if (first + kVec <= width) {
    Unpack(row + first, v);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = first + i < width ? ToFloat(row[first + i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void StoreChunk(T* row, int first, int width, const float (&v)[kVec]) {
  T t[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) t[i] = FromFloat<T>(v[i]);
  if (first + kVec <= width) {
    __builtin_memcpy(row + first, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (first + i < width) row[first + i] = t[i];
  }
}

// ---- one row -----------------------------------------------------------------------------------------------------

struct RowArgs {
  const void* x;
  const void* residual;
  const void* weight;
  int8_t* q;
  float* scale;
  void* sum;
  long long rows;
  long long first_row;  // of this launch
  long long x_stride, residual_stride, q_stride, sum_stride;
  int width;
  int weight_f32;  // the norm's weight: fp32, or the type of x
  double eps;
};

// p of chunk `first`; kNormResidual also writes the sum, rounded to T, and normalises the rounded one
template <typename T, int kMode>
__device__ __forceinline__ void RowChunk(const RowArgs& a, long long row, int first, float (&p)[kVec], double& squares,
                                         bool write_sum) {
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  LoadChunk(x, first, a.width, p);
  if constexpr (kMode == kGate) {
    float up[kVec];
    LoadChunk(x + a.width, first, a.width, up);
#pragma unroll
    for (int i = 0; i < kVec; ++i) p[i] = p[i] / (1.f + expf(-p[i])) * up[i];
  }
  if constexpr (kMode == kNormResidual) {
    float r[kVec];
    LoadChunk(static_cast<const T*>(a.residual) + row * a.residual_stride, first, a.width, r);
#pragma unroll
    for (int i = 0; i < kVec; ++i) p[i] = ToFloat(FromFloat<T>(p[i] + r[i]));
    if (write_sum) StoreChunk(static_cast<T*>(a.sum) + row * a.sum_stride, first, a.width, p);
  }
  if constexpr (kMode == kNorm || kMode == kNormResidual) {
    float w[kVec];
    if (a.weight_f32) LoadChunk(static_cast<const float*>(a.weight), first, a.width, w);
    else LoadChunk(static_cast<const T*>(a.weight), first, a.width, w);
    // squares in 64 bits: they hold for every value of the 32-bit range, where 32-bit squares overflow from 2^64
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      squares = fma(static_cast<double>(p[i]), static_cast<double>(p[i]), squares);
      p[i] *= w[i];
    }
  }
}

__device__ __forceinline__ unsigned AbsBits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

constexpr unsigned kInfBits = 0x7f800000u;

// |p| compared as bit patterns: the order of the magnitudes, with infinity and NaN above every finite value
__device__ __forceinline__ unsigned MaxBits(const float (&p)[kVec], unsigned top) {
#pragma unroll
  for (int i = 0; i < kVec; ++i) top = max(top, AbsBits(p[i]));
  return top;
}

__device__ __attribute__((noinline)) int ExactLevel(float p, float top) {
  return static_cast<int>(rint(127.0 * static_cast<double>(p) / static_cast<double>(top)));
}

// eight integers of a row whose maximum is `top` (finite, not zero) and inverse = 127 / top
__device__ __forceinline__ uint64_t Levels(const float (&p)[kVec], float top, float inverse) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, ties to even, in the low bits
  unsigned level[kVec];
  float worst = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const float t = p[i] * inverse;
    const float shifted = t + kMagic;
    level[i] = __float_as_uint(shifted);
    worst = fmaxf(worst, fabsf(t - (shifted - kMagic)));
  }
  // below 2^-100 the inverse overflows or p loses bits: all of the row in 64 bits
  if (worst > 0.49996f || top < 0x1p-100f) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) level[i] = static_cast<unsigned>(ExactLevel(p[i], top));
  }
  uint64_t packed = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) packed |= static_cast<uint64_t>(level[i] & 0xffu) << (8 * i);
  return packed;
}

__device__ __forceinline__ void StoreLevels(int8_t* row, int first, int width, uint64_t packed) {
  if (first + kVec <= width) {
    __builtin_memcpy(row + first, &packed, sizeof(packed));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (first + i < width) row[first + i] = static_cast<int8_t>(packed >> (8 * i));
  }
}

// the row's maximum and sum of squares over all threads of the row
template <bool kNeedSum, bool kOneWave>
__device__ __forceinline__ void ReduceRow(unsigned& top, double& squares) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    top = max(top, static_cast<unsigned>(__shfl_xor(static_cast<int>(top), d, 64)));
    if constexpr (kNeedSum) squares += __shfl_xor(squares, d, 64);
  }
  if constexpr (!kOneWave) {
    __shared__ unsigned tops[16];
    __shared__ double sums[16];
    const int waves = blockDim.x >> 6;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      tops[wave] = top;
      if constexpr (kNeedSum) sums[wave] = squares;
    }
    __syncthreads();
    top = tops[0];
    if constexpr (kNeedSum) squares = sums[0];
    for (int i = 1; i < waves; ++i) {  // the same order in every thread
      top = max(top, tops[i]);
      if constexpr (kNeedSum) squares += sums[i];
    }
  }
}

template <int kMode>
__device__ __forceinline__ void StoreScale(const RowArgs& a, long long row, unsigned top, double squares) {
  if (top >= kInfBits) {
    a.scale[row] = __uint_as_float(0x7fc00000u);
  } else if constexpr (kMode == kNorm || kMode == kNormResidual) {
    const double factor = 1.0 / sqrt(squares / a.width + a.eps);
    a.scale[row] = static_cast<float>(static_cast<double>(__uint_as_float(top)) * factor / 127.0);
  } else {
    // next to the largest fp32 value 127 s can round to infinity: there s is the next smaller number
    const float s = __uint_as_float(top) / 127.f;
    a.scale[row] = 127.f * s < __uint_as_float(kInfBits) ? s : __uint_as_float(__float_as_uint(s) - 1);
  }
}

// kChunks chunks per thread stay in registers.  kOneWave: a wavefront per row, four rows per block, no barrier;
// otherwise a block per row.
template <typename T, int kMode, int kChunks, bool kOneWave>
__global__ __launch_bounds__(kOneWave ? 256 : 1024) void RowsKernel(RowArgs a) {
  constexpr bool kNeedSum = kMode == kNorm || kMode == kNormResidual;
  const int threads = kOneWave ? 64 : blockDim.x;
  const int t = kOneWave ? (threadIdx.x & 63) : threadIdx.x;
  const long long row = kOneWave ? a.first_row + static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6)
                                 : a.first_row + blockIdx.x;
  if (kOneWave && row >= a.rows) return;
  float p[kChunks][kVec];
  unsigned top = 0;
  double squares = 0.0;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int first = (c * threads + t) * kVec;
    if (first < a.width) {
      RowChunk<T, kMode>(a, row, first, p[c], squares, true);
      top = MaxBits(p[c], top);
    }
  }
  ReduceRow<kNeedSum, kOneWave>(top, squares);
  if (t == 0) StoreScale<kMode>(a, row, top, squares);
  const float largest = __uint_as_float(top);
  const bool live = top != 0 && top < kInfBits;  // the same in the whole row
  const float inverse = 127.f / largest;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int first = (c * threads + t) * kVec;
    if (first < a.width) StoreLevels(q, first, a.width, live ? Levels(p[c], largest, inverse) : 0);
  }
}

// Rows that do not fit into a block's registers: the row is read twice, the second time mostly from L2.  The second
// pass computes p anew from the inputs - except that a sum written over one of them is read back instead.
template <typename T, int kMode>
__global__ __launch_bounds__(1024) void LongRowsKernel(RowArgs a) {
  constexpr bool kNeedSum = kMode == kNorm || kMode == kNormResidual;
  const long long row = a.first_row + blockIdx.x;
  unsigned top = 0;
  double squares = 0.0;
  for (long long at = threadIdx.x; at * kVec < a.width; at += blockDim.x) {
    float p[kVec];
    RowChunk<T, kMode>(a, row, static_cast<int>(at) * kVec, p, squares, true);
    top = MaxBits(p, top);
  }
  ReduceRow<kNeedSum, false>(top, squares);
  if (threadIdx.x == 0) StoreScale<kMode>(a, row, top, squares);
  const float largest = __uint_as_float(top);
  const bool live = top != 0 && top < kInfBits;
  const float inverse = 127.f / largest;
  RowArgs again = a;
  if constexpr (kMode == kNormResidual) {  // each thread reads back what it wrote itself
    again.x = a.sum;
    again.x_stride = a.sum_stride;
  }
  constexpr int kAgain = kMode == kNormResidual ? kNorm : kMode;
  int8_t* q = a.q + row * a.q_stride;
  for (long long at = threadIdx.x; at * kVec < a.width; at += blockDim.x) {
    const int first = static_cast<int>(at) * kVec;
    float p[kVec];
    double unused = 0.0;
    RowChunk<T, kAgain>(again, row, first, p, unused, false);
    StoreLevels(q, first, a.width, live ? Levels(p, largest, inverse) : 0);
  }
}

// out[row][k] = round(q[row][k] * scale[row]); one chunk of eight per thread
template <typename T>
__global__ __launch_bounds__(256) void DequantizeKernel(const int8_t* __restrict__ q, const float* __restrict__ scale,
                                                        T* __restrict__ out, long long rows, int width,
                                                        int chunks_per_row, long long q_stride, long long out_stride) {
  const long long chunks = rows * chunks_per_row;
  for (long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; at < chunks;
       at += static_cast<long long>(gridDim.x) * 256) {
    const long long row = chunks >> 31 ? at / chunks_per_row
                                       : static_cast<unsigned>(at) / static_cast<unsigned>(chunks_per_row);
    const int first = static_cast<int>(at - row * chunks_per_row) * kVec;
    const int8_t* src = q + row * q_stride + first;
    const float s = scale[row];
    uint64_t packed = 0;
    if (first + kVec <= width) {
      __builtin_memcpy(&packed, src, sizeof(packed));
    } else {
      for (int i = 0; first + i < width; ++i)
        packed |= static_cast<uint64_t>(static_cast<uint8_t>(src[i])) << (8 * i);
    }
    float v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = static_cast<float>(static_cast<int8_t>(packed >> (8 * i))) * s;
    StoreChunk(out + row * out_stride, first, width, v);
  }
}

int Status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : -1000 - static_cast<int>(e);
}

// A grid holds fewer than 2^32 threads: rows beyond that go to further launches.
constexpr long long kMostRows = 1ll << 21;

template <typename T, int kMode>
void LaunchRows(RowArgs a, hipStream_t stream) {
  const int chunks = (a.width + kVec - 1) / kVec;
  auto threads = [&](int per_thread) { return dim3(((chunks + per_thread - 1) / per_thread + 63) / 64 * 64); };
  const long long rows = a.rows;
  for (; a.first_row < rows; a.first_row += kMostRows) {
    a.rows = rows - a.first_row < kMostRows ? rows : a.first_row + kMostRows;  // one past the last row of this launch
    const unsigned count = static_cast<unsigned>(a.rows - a.first_row);
    if (chunks <= 64)
      hipLaunchKernelGGL((RowsKernel<T, kMode, 1, true>), dim3((count + 3) / 4), dim3(256), 0, stream, a);
    else if (chunks <= 512)
      hipLaunchKernelGGL((RowsKernel<T, kMode, 1, false>), dim3(count), threads(1), 0, stream, a);
    else if (chunks <= 1024)
      hipLaunchKernelGGL((RowsKernel<T, kMode, 2, false>), dim3(count), threads(2), 0, stream, a);
    else if (chunks <= 4096)
      hipLaunchKernelGGL((RowsKernel<T, kMode, 4, false>), dim3(count), threads(4), 0, stream, a);
    else
      hipLaunchKernelGGL((LongRowsKernel<T, kMode>), dim3(count), dim3(1024), 0, stream, a);
  }
}

template <typename T>
int LaunchMode(int mode, const RowArgs& a, hipStream_t stream) {
  switch (mode) {
    case kPlain: LaunchRows<T, kPlain>(a, stream); break;
    case kNorm: LaunchRows<T, kNorm>(a, stream); break;
    case kNormResidual: LaunchRows<T, kNormResidual>(a, stream); break;
    case kGate: LaunchRows<T, kGate>(a, stream); break;
    default: return -2;
  }
  return Status();
}

// positions within a row are ints, the two halves of a gated one included
bool BadExtent(long long rows, long long width) { return rows <= 0 || width <= 0 || width > (1ll << 30); }

int Rows(int mode, int dtype, const RowArgs& a, void* stream) {
  switch (dtype) {
    case tca::kF32: return LaunchMode<float>(mode, a, static_cast<hipStream_t>(stream));
    case tca::kF16: return LaunchMode<_Float16>(mode, a, static_cast<hipStream_t>(stream));
    case tca::kBF16: return LaunchMode<Bf16>(mode, a, static_cast<hipStream_t>(stream));
    default: return -2;
  }
}

}  // namespace

extern "C" {

int tca_int8_quantize_launch(const void* x, void* q, void* scale, int dtype, int gated, long long rows, long long width,
                             long long x_stride, long long q_stride, void* stream) {
  if (!x || !q || !scale || BadExtent(rows, width)) return -1;
  RowArgs a{};
  a.x = x;
  a.q = static_cast<int8_t*>(q);
  a.scale = static_cast<float*>(scale);
  a.rows = rows;
  a.width = static_cast<int>(width);
  a.x_stride = x_stride;
  a.q_stride = q_stride;
  return Rows(gated ? kGate : kPlain, dtype, a, stream);
}

int tca_int8_rms_norm_launch(const void* x, const void* residual, const void* weight, void* q, void* scale, void* sum,
                             int dtype, int weight_f32, double eps, long long rows, long long width, long long x_stride,
                             long long residual_stride, long long q_stride, long long sum_stride, void* stream) {
  if (!x || !weight || !q || !scale || BadExtent(rows, width) || (!residual) != (!sum) || !(eps > 0)) return -1;
  RowArgs a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.q = static_cast<int8_t*>(q);
  a.scale = static_cast<float*>(scale);
  a.sum = sum;
  a.rows = rows;
  a.width = static_cast<int>(width);
  a.x_stride = x_stride;
  a.residual_stride = residual_stride;
  a.q_stride = q_stride;
  a.sum_stride = sum_stride;
  a.weight_f32 = weight_f32;
  a.eps = eps;
  return Rows(residual ? kNormResidual : kNorm, dtype, a, stream);
}

int tca_int8_dequantize_launch(const void* q, const void* scale, void* out, int dtype, long long rows, long long width,
                               long long q_stride, long long out_stride, void* stream) {
  if (!q || !scale || !out || BadExtent(rows, width)) return -1;
  const int chunks_per_row = static_cast<int>((width + kVec - 1) / kVec);
  const long long blocks = (rows * chunks_per_row + 255) / 256;
  const dim3 grid(static_cast<unsigned>(blocks < (1ll << 23) ? blocks : 1ll << 23));  // the kernel takes the rest in turns
  const int8_t* src = static_cast<const int8_t*>(q);
  const float* s = static_cast<const float*>(scale);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int w = static_cast<int>(width);
  switch (dtype) {
    case tca::kF32:
      hipLaunchKernelGGL((DequantizeKernel<float>), grid, dim3(256), 0, st, src, s, static_cast<float*>(out), rows, w,
                         chunks_per_row, q_stride, out_stride);
      break;
    case tca::kF16:
      hipLaunchKernelGGL((DequantizeKernel<_Float16>), grid, dim3(256), 0, st, src, s, static_cast<_Float16*>(out), rows, w,
                         chunks_per_row, q_stride, out_stride);
      break;
    case tca::kBF16:
      hipLaunchKernelGGL((DequantizeKernel<Bf16>), grid, dim3(256), 0, st, src, s, static_cast<Bf16*>(out), rows, w,
                         chunks_per_row, q_stride, out_stride);
      break;
    default: return -2;
  }
  return Status();
}

}  // extern "C"
