// Matrix product in 8-bit integers with a scale per token and per output channel (gfx950):
//
//   Y[m][n] = round( (sum_k X[m][k] W[n][k]) sx[m] sw[n] + bias[n] + R[m][n] )
//
// The sum is held in int32 and exact (k <= 131071: 128 * 128 * k stays below 2^31), so its order does not matter and
// no split of k changes a result.  Scales, bias and residual are applied to it in fp32, once, and the result is rounded
// once to the output's type.
//
// Both operands have k contiguous, so an MFMA fragment (v_mfma_i32_16x16x64_i8: 16 rows x 64 k, 16 bytes per lane) is a
// plain 16-byte read.  Which of the 64 k a lane's bytes stand for is the same for both operands, so any assignment of k
// to lanes gives the same sum.  The weight is the MFMA's first operand: a lane then holds four consecutive outputs of
// one token.
//
// SplitKernel  the waves of a block share the k axis of one small output tile: every wave multiplies its own k steps of
//              128 straight from memory to registers, the partial sums meet in LDS.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace {

using int4v = __attribute__((ext_vector_type(4))) int;

struct LinearArgs {
  const int8_t* x;
  const float* x_scale;
  const int8_t* w;
  const float* w_scale;
  const void* bias;      // [n] in the output's type, or null
  const void* residual;  // [m][n] in the output's type, or null
  void* y;
  long long m, n;
  long long x_stride, w_stride, residual_stride, y_stride;
  int k;
  int dtype;
};

__device__ __forceinline__ float Load(const void* p, long long at, int dtype) {
  if (dtype == tca::kF32) return static_cast<const float*>(p)[at];
  if (dtype == tca::kF16) return static_cast<float>(static_cast<const _Float16*>(p)[at]);
  return __uint_as_float(static_cast<unsigned>(static_cast<const unsigned short*>(p)[at]) << 16);
}

__device__ __forceinline__ void Store(void* p, long long at, int dtype, float v) {
  if (dtype == tca::kF32) static_cast<float*>(p)[at] = v;
  else if (dtype == tca::kF16) static_cast<_Float16*>(p)[at] = static_cast<_Float16>(v);
  else static_cast<unsigned short*>(p)[at] = __builtin_bit_cast(unsigned short, static_cast<__bf16>(v));
}

// one lane's accumulators: outputs n .. n + 3 of token m
__device__ __forceinline__ void Finish(const LinearArgs& a, long long m, long long n, int4v acc) {
  if (m >= a.m) return;
  const float sx = a.x_scale[m];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.n) return;
    float v = static_cast<float>(acc[i]) * (sx * a.w_scale[n + i]);
    if (a.bias) v += Load(a.bias, n + i, a.dtype);
    if (a.residual) v += Load(a.residual, m * a.residual_stride + n + i, a.dtype);
    Store(a.y, m * a.y_stride + n + i, a.dtype, v);
  }
}

// 16 bytes of a row from k on; zeros past the row's end (bytes there may belong to nobody)
__device__ __forceinline__ int4v LoadTail(const int8_t* row, int k, int end) {
  int4v v = {0, 0, 0, 0};
  if (k + 16 <= end) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    unsigned char bytes[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) bytes[i] = k + i < end ? static_cast<unsigned char>(row[k + i]) : 0;
    __builtin_memcpy(&v, bytes, 16);
  }
  return v;
}

constexpr int kStep = 128;  // k per wave and step: a lane reads 32 consecutive bytes, four lanes a whole cache line

// Block tile: 16 kMT tokens x 16 kNT outputs, k split over kWaves waves.
template <int kMT, int kNT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void SplitKernel(LinearArgs a, long long m_first, unsigned tiles_n) {
  extern __shared__ __attribute__((aligned(16))) int4v parts[];  // [kWaves][kMT * kNT][64]
  const unsigned tile_m = blockIdx.x / tiles_n;
  const unsigned tile_n = blockIdx.x - tile_m * tiles_n;
  const long long m0 = m_first + static_cast<long long>(tile_m) * (16 * kMT);
  const long long n0 = static_cast<long long>(tile_n) * (16 * kNT);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int8_t* xr[kMT];
  const int8_t* wr[kNT];
#pragma unroll
  for (int i = 0; i < kMT; ++i) {  // rows past the end read the last one; their results are not stored
    const long long m = m0 + i * 16 + (lane & 15);
    xr[i] = a.x + (m < a.m ? m : a.m - 1) * a.x_stride;
  }
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    const long long n = n0 + i * 16 + (lane & 15);
    wr[i] = a.w + (n < a.n ? n : a.n - 1) * a.w_stride;
  }
  int4v acc[kMT][kNT];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) acc[i][j] = int4v{0, 0, 0, 0};
  const int whole = a.k / kStep;
  const int at = (lane >> 4) * 32;
  for (int s = wave; s < whole; s += kWaves) {
    int4v x[kMT][2], w[kNT][2];
#pragma unroll
    for (int j = 0; j < kNT; ++j) __builtin_memcpy(w[j], wr[j] + s * kStep + at, 32);
#pragma unroll
    for (int i = 0; i < kMT; ++i) __builtin_memcpy(x[i], xr[i] + s * kStep + at, 32);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j][h], x[i][h], acc[i][j], 0, 0, 0);
  }
  if (whole * kStep < a.k && wave == whole % kWaves) {  // the last, partial step
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = whole * kStep + at + h * 16;
      int4v x[kMT], w[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) w[j] = LoadTail(wr[j], k, a.k);
#pragma unroll
      for (int i = 0; i < kMT; ++i) x[i] = LoadTail(xr[i], k, a.k);
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x[i], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) parts[(wave * (kMT * kNT) + i * kNT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < kMT * kNT; f += kWaves) {
    int4v sum = parts[f * 64 + lane];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) sum += parts[(v * (kMT * kNT) + f) * 64 + lane];
    Finish(a, m0 + (f / kNT) * 16 + (lane & 15), n0 + (f % kNT) * 16 + (lane >> 4) * 4, sum);
  }
}

int Status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : -1000 - static_cast<int>(e);
}

// A grid holds fewer than 2^32 threads: tokens beyond that go to further launches.
template <int kMT, int kNT, int kWaves>
int LaunchSplit(const LinearArgs& a, hipStream_t stream) {
  const long long tiles_n = (a.n + 16 * kNT - 1) / (16 * kNT);
  constexpr long long kMostBlocks = (1ll << 31) / (64 * kWaves);
  if (tiles_n > kMostBlocks) return -3;
  const long long most_m = kMostBlocks / tiles_n * (16 * kMT);
  for (long long m = 0; m < a.m; m += most_m) {
    const long long left = a.m - m < most_m ? a.m - m : most_m;
    const long long blocks = (left + 16 * kMT - 1) / (16 * kMT) * tiles_n;
    hipLaunchKernelGGL((SplitKernel<kMT, kNT, kWaves>), dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves),
                       kWaves * kMT * kNT * 1024, stream, a, m, static_cast<unsigned>(tiles_n));
  }
  return Status();
}

}  // namespace

extern "C" int tca_int8_linear_launch(const void* x, const void* x_scale, const void* w, const void* w_scale, const void* bias,
                                      const void* residual, void* y, int dtype, long long m, long long n, long long k,
                                      long long x_stride, long long w_stride, long long residual_stride,
                                      long long y_stride, void* stream) {
  if (!x || !x_scale || !w || !w_scale || !y || m <= 0 || n <= 0 || k <= 0) return -1;
  if (dtype != tca::kF32 && dtype != tca::kF16 && dtype != tca::kBF16) return -2;
  if (k > 131071) return -3;
  LinearArgs a{static_cast<const int8_t*>(x),  static_cast<const float*>(x_scale), static_cast<const int8_t*>(w),
               static_cast<const float*>(w_scale), bias, residual, y, m, n, x_stride, w_stride, residual_stride, y_stride,
               static_cast<int>(k), dtype};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return m <= 16 ? LaunchSplit<1, 1, 8>(a, st) : LaunchSplit<4, 4, 4>(a, st);
}
