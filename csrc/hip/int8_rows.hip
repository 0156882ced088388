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

template <typename T>
struct Chunk {  // as it lies in memory
  static constexpr int kWords = 2 * sizeof(T);
  unsigned raw[kWords];
};

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(_Float16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float ToFloat(Bf16 v) { return __uint_as_float(static_cast<unsigned>(v.bits) << 16); }

template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 FromFloat<_Float16>(float v) {
  asm("" : "+v"(v));  // rounded to fp32 first, also where an instruction would round a product to fp16 at once
  return static_cast<_Float16>(v);
}
template <> __device__ __forceinline__ Bf16 FromFloat<Bf16>(float v) {
  return Bf16{__builtin_bit_cast(unsigned short, static_cast<__bf16>(v))};  // nearest, ties to even, NaN kept
}

// The chunk at `first`.  Where the row ends inside it, its last eight values instead; behind the row's end, values that
// are not used.  No branch: all requests of a thread are on their way before it waits for one.  Rows shorter than a
// chunk (kShort) are read one by one.
template <bool kShort, typename T>
__device__ __forceinline__ Chunk<T> Request(const T* row, int first, int width) {
  Chunk<T> c;
  if constexpr (!kShort) {
    __builtin_memcpy(&c, row + min(first, width - kVec), sizeof(c));
  } else {
    T t[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) t[i] = i < width ? row[i] : T{};
    __builtin_memcpy(&c, t, sizeof(c));
  }
  return c;
}

// Its values, zeros behind the row's end
template <bool kShort, typename T>
__device__ __forceinline__ void Values(Chunk<T> c, int first, int width, float (&v)[kVec]) {
  constexpr int kWords = Chunk<T>::kWords;
  const int past = first + kVec - width;  // values that belong to the chunk before this one
  if (!kShort && past > 0) {              // they are moved out
#pragma unroll
    for (int step = 4; step >= 1; step /= 2) {
      if (past & step) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          if constexpr (sizeof(T) == 2) {
            if (step == 1) c.raw[i] = c.raw[i] >> 16 | (i + 1 < kWords ? c.raw[i + 1] << 16 : 0u);
            else c.raw[i] = i + step / 2 < kWords ? c.raw[i + step / 2] : 0u;
          } else {
            c.raw[i] = i + step < kWords ? c.raw[i + step] : 0u;
          }
        }
      }
    }
  }
  T t[kVec];
  __builtin_memcpy(t, &c, sizeof(t));
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = ToFloat(t[i]);
}

// N bytes to any address, by non-temporal stores: what a kernel writes does not push out what it and its neighbours are
// still to read (norm and read-back of 16384 x 8192: 240 -> 229 us, the norm alone of 2048 x 8192 28.8 -> 22.4; a reader
// that follows at once finds small results no later, 36.3 and 36.4 us for that norm and its read-back).  Not where a lane
// has 32 bytes: each of its stores leaves gaps between the lanes, to be filled by the next, and that needs the caches.
template <int N>
__device__ __forceinline__ void StoreBytes(void* to, const void* from) {
  using Word = __attribute__((ext_vector_type(N >= 16 ? 4 : 2))) unsigned;
  typedef Word AnyAddress __attribute__((aligned(1)));
#pragma unroll
  for (int i = 0; i < N / static_cast<int>(sizeof(Word)); ++i) {
    Word w;
    __builtin_memcpy(&w, static_cast<const char*>(from) + i * sizeof(Word), sizeof(Word));
    AnyAddress* const at = reinterpret_cast<AnyAddress*>(static_cast<char*>(to) + i * sizeof(Word));
    if constexpr (N == sizeof(Word)) __builtin_nontemporal_store(w, at);
    else *at = w;
  }
}

template <typename T, int kCount>
__device__ __forceinline__ void StoreChunk(T* row, int first, int width, const float (&v)[kCount]) {
  T t[kCount];
#pragma unroll
  for (int i = 0; i < kCount; ++i) t[i] = FromFloat<T>(v[i]);
  if (first + kCount <= width) {
    StoreBytes<sizeof(t)>(row + first, t);
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
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
  double eps, inverse_width;
};

// g / (1 + exp(-g)), within 7 half steps of fp32 (2^-24).  With z = exp(-|g|) <= 1 it is g / (1 + z) or g z / (1 + z), in
// which nothing overflows.  z = 2^n 2^f for the integer n nearest to -|g| log2 e: f is that product less n in fused steps
// with log2 e in two parts, 2^f comes from the unit; the quotient from the unit's reciprocal and one correction.  16
// instructions where the library's exp and division take about 40, and the kernel was bound by them.
__device__ __forceinline__ float Silu(float g) {
  constexpr float kLog2E = 0x1.715476p+0f, kLog2ELow = 0x1.4ae0cp-26f;
  const float a = -fminf(fabsf(g), 200.f);  // exp(-200) is 0 in fp32
  const float n = rintf(a * kLog2E);
  const float f = fmaf(a, kLog2ELow, fmaf(a, kLog2E, -n));
  const float z = ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n));
  const float d = 1.f + z, r = __builtin_amdgcn_rcpf(d);
  const float over = g < 0.f ? g * z : g;
  const float y = over * r;
  return fmaf(fmaf(-y, d, over), r, y);
}

// What a chunk of p is made from: x; the other factor, or the residual; the weight, of type W
template <typename T, typename W>
struct Inputs {
  Chunk<T> x, second;
  Chunk<W> weight;
};

template <typename T>
__device__ __forceinline__ const T* Row(const void* p, long long row, long long stride) {
  return static_cast<const T*>(p) + row * stride;
}

template <typename T, typename W, int kMode, bool kShort>
__device__ __forceinline__ Inputs<T, W> RequestInputs(const RowArgs& a, long long row, int first) {
  Inputs<T, W> in;
  const T* x = Row<T>(a.x, row, a.x_stride);
  in.x = Request<kShort>(x, first, a.width);
  if constexpr (kMode == kGate) in.second = Request<kShort>(x + a.width, first, a.width);
  if constexpr (kMode == kNormResidual) in.second = Request<kShort>(Row<T>(a.residual, row, a.residual_stride), first, a.width);
  if constexpr (kMode == kNorm || kMode == kNormResidual) in.weight = Request<kShort>(static_cast<const W*>(a.weight), first, a.width);
  return in;
}

// p of chunk `first`; kNormResidual also writes the sum, rounded to T, and normalises the rounded one
template <typename T, typename W, int kMode, bool kShort>
__device__ __forceinline__ void RowChunk(const RowArgs& a, long long row, int first, const Inputs<T, W>& in,
                                         float (&p)[kVec], double& squares) {
  Values<kShort>(in.x, first, a.width, p);
  if constexpr (kMode == kGate) {
    float up[kVec];
    Values<kShort>(in.second, first, a.width, up);
#pragma unroll
    for (int i = 0; i < kVec; ++i) p[i] = Silu(p[i]) * up[i];
  }
  if constexpr (kMode == kNormResidual) {
    float r[kVec];
    Values<kShort>(in.second, first, a.width, r);
#pragma unroll
    for (int i = 0; i < kVec; ++i) p[i] = ToFloat(FromFloat<T>(p[i] + r[i]));
    StoreChunk(static_cast<T*>(a.sum) + row * a.sum_stride, first, a.width, p);
  }
  if constexpr (kMode == kNorm || kMode == kNormResidual) {
    float w[kVec];
    Values<kShort>(in.weight, first, a.width, w);
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
    const float shifted = fmaf(p[i], inverse, kMagic);
    level[i] = __float_as_uint(shifted);
    worst = fmaxf(worst, fabsf(fmaf(p[i], inverse, kMagic - shifted)));
  }
  // below 2^-100 the inverse overflows or p loses bits: all of the row in 64 bits
  if (worst > 0.49996f || top < 0x1p-100f) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) level[i] = static_cast<unsigned>(ExactLevel(p[i], top));
  }
  unsigned half[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)  // the low bytes of four
    half[h] = __builtin_amdgcn_perm(level[4 * h + 1], level[4 * h], 0x0c0c0400u) |
              __builtin_amdgcn_perm(level[4 * h + 3], level[4 * h + 2], 0x04000c0cu);
  return half[0] | static_cast<uint64_t>(half[1]) << 32;
}

__device__ __forceinline__ void StoreLevels(int8_t* row, int first, int width, uint64_t packed) {
  if (first + kVec <= width) {
    StoreBytes<sizeof(packed)>(row + first, &packed);
  } else {
#pragma unroll
    for (int i = 0; i < kVec - 1; ++i)
      if (first + i < width) row[first + i] = static_cast<int8_t>(packed >> (8 * i));
  }
}

// v of the lanes that step s of a reduction over the wave puts together: within rows of 16 lanes through the data path's
// own permutations, then by exchanging rows.  The same pair in the same order, or its mirror image, in both lanes.
template <int kStep>
__device__ __forceinline__ void Pair(unsigned v, unsigned& first, unsigned& second) {
  if constexpr (kStep < 4) {
    constexpr int kPermutation[] = {0xB1, 0x4E, 0x141, 0x140};  // lanes 1 0 3 2, 2 3 0 1, half rows and rows mirrored
    first = v;
    second = __builtin_amdgcn_update_dpp(0, v, kPermutation[kStep], 0xf, 0xf, true);
  } else if constexpr (kStep == 4) {
    const auto swapped = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    first = swapped[0];
    second = swapped[1];
  } else {
    const auto swapped = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    first = swapped[0];
    second = swapped[1];
  }
}

template <bool kNeedSum, int kSteps = 6, int kStep = 0>
__device__ __forceinline__ void ReduceWave(unsigned& top, double& squares) {  // over 2^kSteps neighbouring lanes
  if constexpr (kStep < kSteps) {
    unsigned first, second;
    Pair<kStep>(top, first, second);
    top = max(first, second);
    if constexpr (kNeedSum) {
      const uint64_t bits = __builtin_bit_cast(uint64_t, squares);
      unsigned low[2], high[2];
      Pair<kStep>(static_cast<unsigned>(bits), low[0], low[1]);
      Pair<kStep>(static_cast<unsigned>(bits >> 32), high[0], high[1]);
      squares = __builtin_bit_cast(double, low[0] | static_cast<uint64_t>(high[0]) << 32) +
                __builtin_bit_cast(double, low[1] | static_cast<uint64_t>(high[1]) << 32);
    }
    ReduceWave<kNeedSum, kSteps, kStep + 1>(top, squares);
  }
}

// the row's maximum and sum of squares over all threads of the row
template <bool kNeedSum>
__device__ __forceinline__ void ReduceRow(unsigned& top, double& squares) {
  ReduceWave<kNeedSum>(top, squares);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return;
  __shared__ unsigned tops[16];
  __shared__ double sums[16];
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

template <int kMode>
__device__ __forceinline__ void StoreScale(const RowArgs& a, long long row, unsigned top, double squares) {
  if (top >= kInfBits) {
    a.scale[row] = __uint_as_float(0x7fc00000u);
  } else if constexpr (kMode == kNorm || kMode == kNormResidual) {
    const double mean = fma(squares, a.inverse_width, a.eps);
    double factor = 1.0;
    if (mean > 0x1p-1000) {  // the unit's 24 bits and a step of third order
      factor = __builtin_amdgcn_rsq(mean);
      const double off = fma(-mean * factor, factor, 1.0);
      factor = fma(factor * off, fma(0.375, off, 0.5), factor);
    } else {
      factor = 1.0 / sqrt(mean);
    }
    a.scale[row] = static_cast<float>(static_cast<double>(__uint_as_float(top)) * factor * (1.0 / 127.0));
  } else {
    // next to the largest fp32 value 127 s can round to infinity: there s is the next smaller number
    const float s = __uint_as_float(top) / 127.f;
    a.scale[row] = 127.f * s < __uint_as_float(kInfBits) ? s : __uint_as_float(__float_as_uint(s) - 1);
  }
}

// p of kChunks chunks in registers, the maximum and the sum of this thread's
template <typename T, typename W, int kMode, int kChunks, bool kShort>
__device__ __forceinline__ void TakeRow(const RowArgs& a, long long row, int t, int threads, float (&p)[kChunks][kVec],
                                        unsigned& top, double& squares) {
  Inputs<T, W> in[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) in[c] = RequestInputs<T, W, kMode, kShort>(a, row, (c * threads + t) * kVec);
  top = 0;
  squares = 0.0;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int first = (c * threads + t) * kVec;
    if (first < a.width) {
      RowChunk<T, W, kMode, kShort>(a, row, first, in[c], p[c], squares);
      top = MaxBits(p[c], top);
    }
  }
}

template <int kMode, int kChunks>
__device__ __forceinline__ void GiveRow(const RowArgs& a, long long row, int t, int threads, const float (&p)[kChunks][kVec],
                                        unsigned top, double squares) {
  const float largest = __uint_as_float(top);
  const bool live = top != 0 && top < kInfBits;  // the same in the whole row
  const float inverse = 127.f / largest;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int first = (c * threads + t) * kVec;
    if (first < a.width) StoreLevels(q, first, a.width, live ? Levels(p[c], largest, inverse) : 0);
  }
  if (t == 0) StoreScale<kMode>(a, row, top, squares);
}

// A block per row, kChunks chunks per thread.
template <typename T, typename W, int kMode, int kChunks>
__global__ __launch_bounds__(1024) void RowsKernel(RowArgs a) {
  const long long row = a.first_row + blockIdx.x;
  float p[kChunks][kVec];
  unsigned top;
  double squares;
  TakeRow<T, W, kMode, kChunks, false>(a, row, threadIdx.x, blockDim.x, p, top, squares);
  ReduceRow<kMode == kNorm || kMode == kNormResidual>(top, squares);
  GiveRow<kMode>(a, row, threadIdx.x, blockDim.x, p, top, squares);
}

// Rows of at most 8, 16 or 32 chunks: 2^kSteps lanes per row, 256 threads per block.
template <typename T, typename W, int kMode, int kSteps, bool kShort>
__global__ __launch_bounds__(256) void NarrowRowsKernel(RowArgs a) {
  constexpr int kLanes = 1 << kSteps;
  const long long row = a.first_row + static_cast<long long>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  const int t = threadIdx.x % kLanes;
  if (row >= a.rows) return;
  float p[1][kVec];
  unsigned top;
  double squares;
  TakeRow<T, W, kMode, 1, kShort>(a, row, t, kLanes, p, top, squares);
  ReduceWave<kMode == kNorm || kMode == kNormResidual, kSteps>(top, squares);
  GiveRow<kMode>(a, row, t, kLanes, p, top, squares);
}

// Rows that do not fit into a block's registers: the row is read twice, the second time mostly from L2.  The second
// pass computes p anew from the inputs; a sum, which may lie over one of them, is read back instead.
template <typename T, typename W, int kMode>
__global__ __launch_bounds__(1024) void LongRowsKernel(RowArgs a) {
  constexpr bool kNeedSum = kMode == kNorm || kMode == kNormResidual;
  const long long row = a.first_row + blockIdx.x;
  unsigned top = 0;
  double squares = 0.0;
  for (long long at = threadIdx.x; at * kVec < a.width; at += blockDim.x) {
    const int first = static_cast<int>(at) * kVec;
    float p[kVec];
    RowChunk<T, W, kMode, false>(a, row, first, RequestInputs<T, W, kMode, false>(a, row, first), p, squares);
    top = MaxBits(p, top);
  }
  ReduceRow<kNeedSum>(top, squares);
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
    RowChunk<T, W, kAgain, false>(again, row, first, RequestInputs<T, W, kAgain, false>(again, row, first), p, unused);
    StoreLevels(q, first, a.width, live ? Levels(p, largest, inverse) : 0);
  }
}

// out[row][k] = round(q[row][k] * scale[row]); a thread has 16 bytes of results, so that a wave's store fills whole lines
// (fp32 of 8192 x 8192: with 32 bytes a thread 98 us, or 60 through the caches).
template <typename T>
__global__ __launch_bounds__(256) void DequantizeKernel(const int8_t* __restrict__ q, const float* __restrict__ scale,
                                                        T* __restrict__ out, long long rows, int width,
                                                        int chunks_per_row, long long q_stride, long long out_stride) {
  constexpr int kCount = 16 / sizeof(T);
  const long long chunks = rows * chunks_per_row;
  for (long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; at < chunks;
       at += static_cast<long long>(gridDim.x) * 256) {
    const long long row = chunks >> 31 ? at / chunks_per_row
                                       : static_cast<unsigned>(at) / static_cast<unsigned>(chunks_per_row);
    const int first = static_cast<int>(at - row * chunks_per_row) * kCount;
    const int8_t* src = q + row * q_stride + first;
    const float s = scale[row];
    uint64_t packed = 0;
    if (first + kCount <= width) {
      __builtin_memcpy(&packed, src, kCount);
    } else {
      for (int i = 0; first + i < width; ++i)
        packed |= static_cast<uint64_t>(static_cast<uint8_t>(src[i])) << (8 * i);
    }
    float v[kCount];
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = static_cast<float>(static_cast<int8_t>(packed >> (8 * i))) * s;
    StoreChunk(out + row * out_stride, first, width, v);
  }
}

int Status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : -1000 - static_cast<int>(e);
}

// A grid holds fewer than 2^32 threads: rows beyond that go to further launches.
constexpr long long kMostRows = 1ll << 21;

// Few rows: as many threads as a row has chunks, every chunk's way from memory at the same time (8 rows of 8192 bf16: 5.0
// us with one chunk per thread, 7.0 with four).  Many rows fill the CUs anyway, and what counts is the bytes that a thread
// has on their way: 64 do best, 32 where each CU has few rows.  Times with one, two and four chunks per thread, bf16 from
// memory: 16384 rows of 8192 quantised 120, 87 and 74 us (16 bytes of input a chunk), the norm with a residual 184, 169 and
// 172, the gate 138, 125 and 122 (32 bytes); 2048 rows of 4096 10.6, 9.9 and 11.0; 16.0, 17.4 and 19.0; 12.3, 12.2 and 13.6.
// The gate keeps to two: four, in blocks of 512 threads, gain little where they fill the block (4096 rows of 16384: 62.5 us,
// 63.3 with two) and lose where they do not (of 8200 36.6 and 33.0, of 12000 53.3 and 48.0; fp32 rows of 8200 69.4 and 55.5).
// Norms of fp32 rows hold three fp32 inputs per value: two chunks are what the registers of 1024 threads hold.  Of the kernels
// of four, two spill 4 and 8 registers, for rows of more than 16384 values, which would be read twice otherwise: the gate of
// fp32 rows is faster all the same (2048 of 20000 92 and 100 us, of 32768 136 and 164), and the norm with a residual of bf16
// rows and an fp32 weight with few rows (256 of 32768 14.6 and 17.4 us, 2048 of them 125 and 119).
template <typename T, typename W, int kMode>
void LaunchRows(RowArgs a, hipStream_t stream) {
  constexpr bool kWide = sizeof(T) == 4 && (kMode == kNorm || kMode == kNormResidual);
  const int chunks = (a.width + kVec - 1) / kVec;
  const long long rows = a.rows;
  const int most = kWide ? 2 : 4;
  constexpr int kInputs = kMode == kGate || kMode == kNormResidual ? 2 : 1;  // the norm's weight stays in the caches
  const int bytes = rows >= 4096 ? 64 : 32;
  int per_thread = rows >= 1024 && chunks >= 512 ? bytes / (kInputs * kVec * static_cast<int>(sizeof(T))) : 1;
  per_thread = per_thread < 1 ? 1 : per_thread < most ? per_thread : most;
  while (per_thread < most && chunks > per_thread * 1024) per_thread *= 2;
  const dim3 threads(((chunks + per_thread - 1) / per_thread + 63) / 64 * 64);
  for (; a.first_row < rows; a.first_row += kMostRows) {
    const unsigned count = static_cast<unsigned>(rows - a.first_row < kMostRows ? rows - a.first_row : kMostRows);
    const dim3 blocks(count);
    a.rows = a.first_row + count;  // one past the last row of this launch
    if (a.width < kVec)
      hipLaunchKernelGGL((NarrowRowsKernel<T, W, kMode, 3, true>), dim3((count + 31) / 32), dim3(256), 0, stream, a);
    else if (chunks <= 8)
      hipLaunchKernelGGL((NarrowRowsKernel<T, W, kMode, 3, false>), dim3((count + 31) / 32), dim3(256), 0, stream, a);
    else if (chunks <= 16)
      hipLaunchKernelGGL((NarrowRowsKernel<T, W, kMode, 4, false>), dim3((count + 15) / 16), dim3(256), 0, stream, a);
    else if (chunks <= 32)
      hipLaunchKernelGGL((NarrowRowsKernel<T, W, kMode, 5, false>), dim3((count + 7) / 8), dim3(256), 0, stream, a);
    else if (chunks > per_thread * 1024)
      hipLaunchKernelGGL((LongRowsKernel<T, W, kMode>), blocks, dim3(1024), 0, stream, a);
    else if (per_thread == 1)
      hipLaunchKernelGGL((RowsKernel<T, W, kMode, 1>), blocks, threads, 0, stream, a);
    else if (per_thread == 2)
      hipLaunchKernelGGL((RowsKernel<T, W, kMode, 2>), blocks, threads, 0, stream, a);
    else if constexpr (!kWide)
      hipLaunchKernelGGL((RowsKernel<T, W, kMode, 4>), blocks, threads, 0, stream, a);
  }
}

template <typename T>
int LaunchMode(int mode, const RowArgs& a, hipStream_t stream) {
  switch (mode) {
    case kPlain: LaunchRows<T, T, kPlain>(a, stream); break;
    case kNorm: a.weight_f32 ? LaunchRows<T, float, kNorm>(a, stream) : LaunchRows<T, T, kNorm>(a, stream); break;
    case kNormResidual:
      a.weight_f32 ? LaunchRows<T, float, kNormResidual>(a, stream) : LaunchRows<T, T, kNormResidual>(a, stream);
      break;
    case kGate: LaunchRows<T, T, kGate>(a, stream); break;
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
  a.inverse_width = 1.0 / static_cast<double>(width);
  return Rows(residual ? kNormResidual : kNorm, dtype, a, stream);
}

int tca_int8_dequantize_launch(const void* q, const void* scale, void* out, int dtype, long long rows, long long width,
                               long long q_stride, long long out_stride, void* stream) {
  if (!q || !scale || !out || BadExtent(rows, width)) return -1;
  const int count = dtype == tca::kF32 ? 4 : 8;  // values in 16 bytes of results
  const int chunks_per_row = static_cast<int>((width + count - 1) / count);
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
