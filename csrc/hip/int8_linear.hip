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
// SplitDmaKernel  few tokens or small outputs: the waves of a block share the k axis of one small output tile, every wave
//              multiplies its own k steps of 128 from a ring of its own in LDS, filled by DMA; the sums meet in LDS.  Bound
//              by memory: 16 x 32768 x 4096 in 25 to 28 us (4.8 to 5.4 TB/s), 1 x 4096 x 4096 in 4.5 us on the GPU.
// SplitAnyKernel, TileAnyKernel  the same, and tiles of 64 x 64, for rows that do not start at multiples of 16 bytes, through
//              registers.
// TileKernel   large products: tiles of 64 x 64 to 256 x 256 outputs per block of four waves, operands through LDS stages
//              filled by DMA.  8192 x 8192 x 8192 to bf16, one call behind another on real values: 385 us (2.9 POP/s), 423
//              with a residual.  What bounds it is the card's power, so that the time goes with what ran before: 5 calls after
//              a pause 392 and 424, 20 calls 456 and 491, one alone 447 and 456.  On zeros, where nothing toggles, it took 296
//              and 312 on a card that took 371 and 382 on values, and its products alone, fed from registers, 293 us on
//              values and 259 on zeros.  One wave per SIMD with 128 x 128 outputs reads the fewest bytes from LDS per product and won
//              over two waves with 128 x 64 (408 against 420 us at an earlier stage of tuning); products of 16 x 16 x 64
//              touch the accumulators half as often per operation as those of 32 x 32 x 32 and won although they issue
//              twice as often (443 against 476 us, earlier still).
// Every launch is one kernel; a large product whose rows start anywhere is two (PadKernel first).
#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

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
  int pass_weight;  // few tokens: the weight is read once, and is larger than what the caches would keep of it
  int vector_rows;  // 16 bytes of outputs start at a multiple of 16 bytes, in y and the residual, and end with the row
  int line_rows;    // every row of y starts at a whole line
};

struct Bf16 {
  unsigned short bits;
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
  return Bf16{__builtin_bit_cast(unsigned short, static_cast<__bf16>(v))};
}

// The same roundings in every kernel, so that a token's outputs do not depend on the others of its batch.
__device__ __forceinline__ float Result(int sum, float scale, float bias, float residual) {
  return __builtin_fmaf(static_cast<float>(sum), scale, bias) + residual;
}

// one lane's sums: outputs n .. n + 3 of token m
template <typename T>
__device__ __forceinline__ void FinishFour(const LinearArgs& a, long long m, long long n, int4v sum) {
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  };
  const T* bias = static_cast<const T*>(a.bias) + n;
  const T* residual = static_cast<const T*>(a.residual) + m * a.residual_stride + n;
  T* y = static_cast<T*>(a.y) + m * a.y_stride + n;
  const float sx = a.x_scale[m];
  if (a.vector_rows) {  // n % 4 == 0, so all four are there
    const float4 sw = *reinterpret_cast<const float4*>(a.w_scale + n);
    const float scale[4] = {sx * sw.x, sx * sw.y, sx * sw.z, sx * sw.w};
    Four b{}, r{};
    if (a.bias) b = *reinterpret_cast<const Four*>(bias);
    if (a.residual) r = *reinterpret_cast<const Four*>(residual);
    Four out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out.v[i] = FromFloat<T>(Result(sum[i], scale[i], ToFloat(b.v[i]), ToFloat(r.v[i])));
    *reinterpret_cast<Four*>(y) = out;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i >= a.n) return;
      y[i] = FromFloat<T>(Result(sum[i], sx * a.w_scale[n + i], a.bias ? ToFloat(bias[i]) : 0.f, a.residual ? ToFloat(residual[i]) : 0.f));
    }
  }
}

__device__ __forceinline__ void Finish(const LinearArgs& a, long long m, long long n, int4v sum) {
  if (m >= a.m || n >= a.n) return;
  if (a.dtype == tca::kF32) FinishFour<float>(a, m, n, sum);
  else if (a.dtype == tca::kF16) FinishFour<_Float16>(a, m, n, sum);
  else FinishFour<Bf16>(a, m, n, sum);
}

// 16 bytes of a row from k on, in two steps, so that several requests can be on their way.  Where the row ends among them
// its last 16 bytes are requested instead; a row shorter than that is read one by one.
__device__ __forceinline__ int4v RequestPiece(const int8_t* row, int k, int end) {
  uint64_t v[2] = {0, 0};
  if (end >= 16) {
    __builtin_memcpy(v, row + (k + 16 <= end ? k : end - 16), 16);
  } else {
    for (int i = 15; i >= 0; --i) {  // the highest first, shifted up by those below
      v[1] = v[1] << 8 | v[0] >> 56;
      v[0] = v[0] << 8 | (k + i < end ? static_cast<uint8_t>(row[k + i]) : 0u);
    }
  }
  int4v out;
  __builtin_memcpy(&out, v, 16);
  return out;
}

// What was requested, those that lie before k moved out and zeros past the row's end.
__device__ __forceinline__ int4v PieceOf(int4v requested, int k, int end) {
  int past = k + 16 - end;
  if (end < 16 || past <= 0) return requested;
  uint64_t v[2];
  __builtin_memcpy(v, &requested, 16);
  if (past >= 8) {
    v[0] = v[1];
    v[1] = 0;
    past -= 8;
  }
  if (past >= 8) v[0] = 0;
  else if (past > 0) {
    v[0] = v[0] >> (8 * past) | v[1] << (64 - 8 * past);
    v[1] >>= 8 * past;
  }
  int4v out;
  __builtin_memcpy(&out, v, 16);
  return out;
}

constexpr int kStep = 128;  // k per wave and step: a lane reads 32 consecutive bytes, four lanes a whole cache line

// An offset behind every descriptor's end, also with a row's offset added: the DMA writes zeros for it, loads give zeros,
// stores are dropped.  The host keeps the rows of a tile below 2^30 bytes.
constexpr unsigned kOutside = 0x80000000u;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t Descriptor(const void* p, long long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(p ? bytes : 0), 0x00020000);
}

using lds_ptr_t = __attribute__((address_space(3))) void*;

// Wave-wide copy global -> LDS, 16 bytes per lane, to lds + 16 * lane; kPolicy 2: non-temporal
template <int kPolicy = 0>
__device__ __forceinline__ void DmaToLds(__amdgpu_buffer_rsrc_t rsrc, unsigned offset, int8_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, reinterpret_cast<lds_ptr_t>(reinterpret_cast<uintptr_t>(lds)), 16,
                                           static_cast<int>(offset), 0, 0, kPolicy);
}

template <int kFirst, int kLast, typename F>
__device__ __forceinline__ void Unrolled(F&& f) {
  if constexpr (kFirst < kLast) {
    f(std::integral_constant<int, kFirst>{});
    Unrolled<kFirst + 1, kLast>(f);
  }
}

// The waves' sums of a block's tile meet in LDS, each wave's in the place of its own stages, and leave.
template <int kMT, int kNT, int kWaves>
__device__ __forceinline__ void MeetSums(const LinearArgs& a, long long m0, long long n0, int8_t* lds, int wave_bytes, int lane,
                                         int wave, const int4v (&acc)[kMT][kNT]) {
  int4v* parts = reinterpret_cast<int4v*>(lds + wave * wave_bytes);
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) parts[(i * kNT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < kMT * kNT; f += kWaves) {
    int4v sum = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) sum += *reinterpret_cast<const int4v*>(lds + v * wave_bytes + (f * 64 + lane) * 16);
    Finish(a, m0 + (f / kNT) * 16 + (lane & 15), n0 + (f % kNT) * 16 + (lane >> 4) * 4, sum);
  }
}

// Block tile: 16 kMT tokens x 16 kNT outputs, k split over kWaves waves.  Each wave keeps a ring of kStages steps of its own
// in LDS, filled by DMA, whose lanes go along the rows, eight to a 128-byte line.  (Fragments read straight from memory
// have every lane of a quarter wave in another row: each 16 bytes are a cache lookup of their own, and a CU takes in 14
// bytes per cycle however the loads are arranged.)  No barrier until the sums meet.
template <int kMT, int kNT, int kWaves, int kStages>
__global__ __launch_bounds__(64 * kWaves) void SplitDmaKernel(LinearArgs a, long long m_first, unsigned tiles_n) {
  constexpr int kXDma = 2 * kMT, kDma = 2 * (kMT + kNT);  // copies of 8 rows
  constexpr int kStageBytes = kDma * 1024;
  static_assert(kStages * kStageBytes >= kMT * kNT * 1024, "the sums meet in the ring's place");
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const unsigned tile_m = blockIdx.x / tiles_n;
  const unsigned tile_n = blockIdx.x - tile_m * tiles_n;
  const long long m0 = m_first + static_cast<long long>(tile_m) * (16 * kMT);
  const long long n0 = static_cast<long long>(tile_n) * (16 * kNT);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int8_t* const ring = lds + wave * (kStages * kStageBytes);
  const int x_rows = static_cast<int>(a.m - m0 < 16 * kMT ? a.m - m0 : 16 * kMT);
  const int w_rows = static_cast<int>(a.n - n0 < 16 * kNT ? a.n - n0 : 16 * kNT);
  const auto x_rsrc = Descriptor(a.x + m0 * a.x_stride, (x_rows - 1) * a.x_stride + a.k);
  const auto w_rsrc = Descriptor(a.w + n0 * a.w_stride, (w_rows - 1) * a.w_stride + a.k);
  // Copy i brings rows 8 i .. 8 i + 7 of 128 bytes; a row's chunk c lies at place c ^ ((row >> 1) & 7), which keeps the
  // lanes whose fragment reads the banks serve together in different columns.
  const unsigned x_row = static_cast<unsigned>(lane >> 3) * static_cast<unsigned>(a.x_stride);
  const unsigned w_row = static_cast<unsigned>(lane >> 3) * static_cast<unsigned>(a.w_stride);
  const int chunk = (lane & 7) ^ (lane >> 4);  // of even copies; 4 further on (exclusive or) in odd ones
  auto issue = [&](int s, int stage) {
    unsigned k[2];
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const int at = s * kStep + (chunk ^ (4 * odd)) * 16;
      k[odd] = at < a.k ? static_cast<unsigned>(at) : kOutside;
    }
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      int8_t* to = ring + stage * kStageBytes + i * 1024;
      if (i < kXDma) DmaToLds(x_rsrc, x_row + static_cast<unsigned>(i * 8 * a.x_stride) + k[i & 1], to);
      else if (a.pass_weight) DmaToLds<2>(w_rsrc, w_row + static_cast<unsigned>((i - kXDma) * 8 * a.w_stride) + k[i & 1], to);
      else DmaToLds(w_rsrc, w_row + static_cast<unsigned>((i - kXDma) * 8 * a.w_stride) + k[i & 1], to);
    }
  };
  int4v acc[kMT][kNT];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) acc[i][j] = int4v{0, 0, 0, 0};
  const int steps = (a.k + kStep - 1) / kStep;
  const int frag = (lane & 15) * kStep + ((lane >> 4) ^ ((lane >> 1) & 7)) * 16;
  int ahead = wave;
#pragma unroll
  for (int stage = 0; stage < kStages; ++stage, ahead += kWaves) issue(ahead, stage);  // past the end: zeros
  int stage = 0;
  for (int s = wave; s < steps; s += kWaves) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * kDma) : "memory");
    int4v x[kMT][2], w[kNT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int8_t* from = ring + stage * kStageBytes + (frag ^ (h * 64));
#pragma unroll
      for (int i = 0; i < kMT; ++i) x[i][h] = *reinterpret_cast<const int4v*>(from + i * 16 * kStep);
#pragma unroll
      for (int j = 0; j < kNT; ++j) w[j][h] = *reinterpret_cast<const int4v*>(from + (kMT + j) * 16 * kStep);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before it is filled again
    issue(ahead, stage);
    ahead += kWaves;
    stage = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j][h], x[i][h], acc[i][j], 0, 0, 0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  MeetSums<kMT, kNT, kWaves>(a, m0, n0, lds, kStages * kStageBytes, lane, wave, acc);
}

// The same for rows at any address, which the DMA does not take: a step's pieces come to registers along the rows, as the
// DMA's lanes go, and are written to the wave's part of LDS when the step before them has been read.
template <int kMT, int kNT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void SplitAnyKernel(LinearArgs a, long long m_first, unsigned tiles_n) {
  constexpr int kXPieces = 2 * kMT, kPieces = 2 * (kMT + kNT);  // 8 rows of 128 bytes each
  constexpr int kStageBytes = kPieces * 1024;
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const unsigned tile_m = blockIdx.x / tiles_n;
  const unsigned tile_n = blockIdx.x - tile_m * tiles_n;
  const long long m0 = m_first + static_cast<long long>(tile_m) * (16 * kMT);
  const long long n0 = static_cast<long long>(tile_n) * (16 * kNT);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int8_t* const stage = lds + wave * kStageBytes;
  const int chunk = (lane & 7) ^ (lane >> 4);  // as in SplitDmaKernel
  const int8_t* row[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {  // rows past the end read the last one; their results are not stored
    if (i < kXPieces) {
      const long long m = m0 + i * 8 + (lane >> 3);
      row[i] = a.x + (m < a.m ? m : a.m - 1) * a.x_stride;
    } else {
      const long long n = n0 + (i - kXPieces) * 8 + (lane >> 3);
      row[i] = a.w + (n < a.n ? n : a.n - 1) * a.w_stride;
    }
  }
  const int steps = (a.k + kStep - 1) / kStep;
  int4v piece[kPieces];
  auto load = [&](int s) {
    if (s * kStep + kStep <= a.k) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) __builtin_memcpy(&piece[i], row[i] + s * kStep + (chunk ^ (4 * (i & 1))) * 16, 16);
    } else if (s < steps) {  // the row ends in this step
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int k = s * kStep + (chunk ^ (4 * (i & 1))) * 16;
        piece[i] = PieceOf(RequestPiece(row[i], k, a.k), k, a.k);
      }
    }
  };
  int4v acc[kMT][kNT];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) acc[i][j] = int4v{0, 0, 0, 0};
  const int frag = (lane & 15) * kStep + ((lane >> 4) ^ ((lane >> 1) & 7)) * 16;
  load(wave);
  for (int s = wave; s < steps; s += kWaves) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) *reinterpret_cast<int4v*>(stage + i * 1024 + lane * 16) = piece[i];
    load(s + kWaves);
    int4v x[kMT][2], w[kNT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int8_t* from = stage + (frag ^ (h * 64));
#pragma unroll
      for (int i = 0; i < kMT; ++i) x[i][h] = *reinterpret_cast<const int4v*>(from + i * 16 * kStep);
#pragma unroll
      for (int j = 0; j < kNT; ++j) w[j][h] = *reinterpret_cast<const int4v*>(from + (kMT + j) * 16 * kStep);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j][h], x[i][h], acc[i][j], 0, 0, 0);
  }
  MeetSums<kMT, kNT, kWaves>(a, m0, n0, lds, kStageBytes, lane, wave, acc);
}

// 16 bytes of consecutive values as they lie in memory.
template <typename T>
struct Part {
  static constexpr int kValues = 16 / sizeof(T);
  unsigned raw[4] = {};
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i]);
    else return ToFloat(__builtin_bit_cast(T, static_cast<unsigned short>(raw[i / 2] >> (16 * (i & 1)))));
  }
};

using uint4v = __attribute__((ext_vector_type(4))) unsigned;

// Through a descriptor: at multiples of 16 bytes, all inside its range or (offset kOutside) not at all.
template <typename T>
__device__ __forceinline__ Part<T> LoadPart(__amdgpu_buffer_rsrc_t rsrc, unsigned offset) {
  const uint4v raw = __builtin_amdgcn_raw_buffer_load_b128(rsrc, static_cast<int>(offset), 0, 0);
  Part<T> v;
#pragma unroll
  for (int c = 0; c < 4; ++c) v.raw[c] = raw[c];
  return v;
}

// At any address, the first `inside` (may be more, or negative) of them.
template <typename T>
__device__ __forceinline__ Part<T> LoadPart(const T* p, int inside) {
  Part<T> v;
  if (inside >= Part<T>::kValues) {
    __builtin_memcpy(v.raw, p, 16);
  } else {
    T t[Part<T>::kValues] = {};
#pragma unroll
    for (int i = 0; i < Part<T>::kValues - 1; ++i)
      if (i < inside) t[i] = p[i];
    __builtin_memcpy(v.raw, t, 16);
  }
  return v;
}

// ---- TileKernel ---------------------------------------------------------------------------------------------------

// k per stage.  An LDS row of an operand is a whole 128-byte line: the DMA takes in 105 to 130 KB per us and CU when eight
// lanes share a line, and 60 to 70 when four do - and that is what a step's time was.
constexpr int kTileK = 128;

// The tiles of a block: each of the 8 XCDs (consecutive blocks go round them) has a contiguous run of tiles, ordered in
// bands of kBand tile rows, so that the tiles an XCD works on at a time share operands in its L2; its blocks take them
// in turn.
constexpr unsigned kBand = 8;

struct Tiles {
  unsigned rows, columns, run;  // of the whole product; tiles per XCD
};

struct TileCursor {
  unsigned at;  // position in the XCD's run
  long long m0, n0;
  int rows, columns;  // inside the matrix; 0 past the last tile

  template <int BM, int BN>
  __device__ __forceinline__ void Place(const LinearArgs& a, const Tiles& t) {
    const unsigned tile = (blockIdx.x & 7) * t.run + at;
    if (at >= t.run || tile >= t.rows * t.columns) {
      m0 = n0 = rows = columns = 0;
      return;
    }
    const unsigned band = tile / (kBand * t.columns);
    const unsigned in_band = tile - band * kBand * t.columns;
    const unsigned high = min(kBand, t.rows - band * kBand);
    const unsigned column = in_band / high;
    m0 = static_cast<long long>(band * kBand + in_band - column * high) * BM;
    n0 = static_cast<long long>(column) * BN;
    rows = static_cast<int>(a.m - m0 < BM ? a.m - m0 : BM);
    columns = static_cast<int>(a.n - n0 < BN ? a.n - n0 : BN);
  }
};

// acc += w x with the accumulator pinned to the accumulation registers: given the choice, the compiler spreads the
// 256 accumulators of a wave over both register files and copies a third of them back and forth in every step
__device__ __forceinline__ void Mfma(int4v w, int4v x, int4v& acc) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(w), "v"(x));
}

// The compiler does not see matrix instructions inside asm: what it needs between them and ordinary instructions that
// touch the accumulators (16 cycles of the instruction and its write) stands here.
__device__ __forceinline__ void SettleAccumulators() { asm volatile("s_nop 15\n\ts_nop 7"); }
__device__ __forceinline__ void Pin(int4v& acc) { asm volatile("" : "+a"(acc)); }  // ordered with the other asm

// How the rows of outputs and residuals lie: at whole 128-byte lines, at multiples of 16 bytes, at any address.
enum Rows : int { kLines, kPieces, kAny };

// Epilogue of a wave, 16 tokens at a time: the accumulators go through LDS (the wave's own part, so no barrier), after
// which a lane holds 16 bytes of consecutive outputs of a token (fp32: two such parts, half of the wave's columns apart)
// and the lanes of a token cover whole cache lines.
//
// kLines, kPieces: through descriptors, whose range ends the columns and rows of a last tile.  Results that fill whole lines
// are stored past the caches and leave the neighbours' operands and residuals their places there (8192 x 8192 x 8192 with a
// residual 466 -> 427 us); parts of lines cost twice the time that way.  Without a residual kResidual may still be set:
// zeros are added, as for a bias that is not there.
template <typename T, int kRowsAt, bool kResidual, int kMT, int kNT>
__device__ __forceinline__ void FinishWave(const LinearArgs& a, const TileCursor& tile, int m, int n, int8_t* lds, int4v (&acc)[kMT][kNT]) {
  constexpr int kSize = sizeof(T);
  constexpr int kPer = Part<T>::kValues, kParts = 8 / kPer;  // a lane's eight outputs
  constexpr int kLanes = kNT * 2;               // lanes of a token
  constexpr int kRows = 64 / kLanes;            // tokens of one access
  constexpr int kTurns = 16 / kRows;            // accesses for 16 tokens
  constexpr int kTurnMask = kNT * 4 < 16 ? kNT * 4 - 1 : 15;
  constexpr int kHeld = kSize == 2 ? 4 : 2;     // steps of 16 tokens whose residual is requested at once
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // addresses are computed here for every tile: kept from tile to tile they would spill
  const int row = m + lane / kLanes;
  const auto sx_rsrc = Descriptor(a.x_scale + tile.m0, tile.rows * 4ll);
  const T* const residual = kResidual && a.residual ? static_cast<const T*>(a.residual) + tile.m0 * a.residual_stride + tile.n0 : nullptr;
  T* const y = static_cast<T*>(a.y) + tile.m0 * a.y_stride + tile.n0;
  const T* const bias_row = a.bias ? static_cast<const T*>(a.bias) + tile.n0 : nullptr;
  // rows past the end start behind the last byte of the last one
  const auto res_rsrc = Descriptor(residual, ((tile.rows - 1) * a.residual_stride + tile.columns) * kSize);
  const auto y_rsrc = Descriptor(y, ((tile.rows - 1) * a.y_stride + tile.columns) * kSize);
  const unsigned y_pitch = static_cast<unsigned>(a.y_stride) * kSize, res_pitch = static_cast<unsigned>(a.residual_stride) * kSize;
  int column[kParts], inside[kParts];
  unsigned y_at[kParts], res_at[kParts];
  float sw[8];
  Part<T> bias[kParts];
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    column[p] = n + (p * kLanes + lane % kLanes) * kPer;
    inside[p] = tile.columns - column[p];
    if constexpr (kRowsAt != kAny) {
      y_at[p] = inside[p] > 0 ? row * y_pitch + column[p] * kSize : kOutside;
      res_at[p] = inside[p] > 0 ? row * res_pitch + column[p] * kSize : kOutside;
      const auto sw_rsrc = Descriptor(a.w_scale + tile.n0, tile.columns * 4ll);
      bias[p] = LoadPart<T>(Descriptor(bias_row, tile.columns * kSize), column[p] * kSize);
#pragma unroll
      for (int c = 0; c < kPer; c += 4) {
        const Part<float> four = LoadPart<float>(sw_rsrc, (column[p] + c) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) sw[p * kPer + c + e] = four[e];
      }
    } else {
      bias[p] = LoadPart(bias_row + column[p], bias_row ? inside[p] : 0);
#pragma unroll
      for (int c = 0; c < kPer; c += 4) {
        const Part<float> four = LoadPart(a.w_scale + tile.n0 + column[p] + c, inside[p] - c);
#pragma unroll
        for (int e = 0; e < 4; ++e) sw[p * kPer + c + e] = four[e];
      }
    }
  }
  const bool ragged = kRowsAt == kAny && tile.columns % kPer != 0;  // some lane's part ends inside its 16 bytes
  float sx[kMT][kTurns];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int t = 0; t < kTurns; ++t)
      sx[i][t] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sx_rsrc, (row + i * 16 + t * kRows) * 4, 0, 0));
  const int write = (lane & 15) * (kNT * 64);
#pragma unroll
  for (int first = 0; first < kMT; first += kHeld) {
    Part<T> r[kHeld][kTurns][kParts];
    if constexpr (kResidual) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
#pragma unroll
        for (int t = 0; t < kTurns; ++t)
#pragma unroll
          for (int p = 0; p < kParts; ++p)
            if (first + i < kMT) {
              const int past = (first + i) * 16 + t * kRows;  // rows from the lane's first
              if constexpr (kRowsAt != kAny) {
                r[i][t][p] = LoadPart<T>(res_rsrc, res_at[p] + past * res_pitch);
              } else if (residual) {
                // rows and parts past the end read others, whose sums are not stored; no branch, so all are on their way
                const char* from = reinterpret_cast<const char*>(residual) + min(row + past, tile.rows - 1) * res_pitch;
                if (tile.columns >= kPer) __builtin_memcpy(r[i][t][p].raw, from + (inside[p] >= kPer ? column[p] * kSize : 0), 16);
                if (ragged && inside[p] < kPer) r[i][t][p] = LoadPart(reinterpret_cast<const T*>(from) + column[p], inside[p]);
              }
            }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = first; i < first + kHeld && i < kMT; ++i) {
#pragma unroll
      for (int j = 0; j < kNT; ++j)
        *reinterpret_cast<int4v*>(lds + write + ((j * 4 + (lane >> 4)) ^ (lane & kTurnMask)) * 16) = acc[i][j];
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int from = lane / kLanes + t * kRows;
        const int past = i * 16 + t * kRows;
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          T v[kPer];
#pragma unroll
          for (int c = 0; c < kPer; c += 4) {
            const int at = kParts == 1 ? lane % kLanes * 2 + c / 4 : p * kLanes + lane % kLanes;
            const int4v sum = *reinterpret_cast<const int4v*>(lds + from * (kNT * 64) + (at ^ (from & kTurnMask)) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float scale = sx[i][t] * sw[p * kPer + c + e];
              float residual_value = 0.f;
              if constexpr (kResidual) residual_value = r[i - first][t][p][c + e];
              v[c + e] = FromFloat<T>(Result(sum[e], scale, bias[p][c + e], residual_value));
            }
          }
          if constexpr (kRowsAt != kAny) {
            uint4v raw;
            __builtin_memcpy(&raw, v, 16);
            __builtin_amdgcn_raw_buffer_store_b128(raw, y_rsrc, static_cast<int>(y_at[p] + past * y_pitch), 0,
                                                   kRowsAt == kLines ? 2 : 0);  // 2: non-temporal
          } else if (row + past < tile.rows) {
            T* const to = reinterpret_cast<T*>(reinterpret_cast<char*>(y) + static_cast<unsigned>(row + past) * y_pitch) + column[p];
            if (inside[p] >= kPer) __builtin_memcpy(to, v, 16);
            asm volatile("");  // or the two kinds of stores are merged, into many small ones
            if (ragged && inside[p] < kPer) {
#pragma unroll
              for (int c = 0; c < kPer - 1; ++c)
                if (c < inside[p]) to[c] = v[c];
            }
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // registers: no more than 16 tokens at a time
    }
  }
}

// A block keeps a ring of kStages stages, each 128 k of a BM x BN tile's operands, and works through its tiles as one
// sequence of stages: the first stages of the next tile are on their way while this one is finished.
//
// A stage's two halves of 64 k are multiplied from registers.  While the second half of one is, both halves of the next are
// read, so that its place in LDS is free for the DMA a whole stage before its products end: with two stages in LDS a request
// has the time of one to one and a half stages to arrive.  That takes a third set of fragment registers: the first halves
// have one, the second halves two in turn.
template <typename T, int BM, int BN, int kWM, int kWN, int kStages, int kBlocks>
__global__ __launch_bounds__(64 * kWM * kWN, kBlocks) void TileKernel(LinearArgs a, Tiles tiles) {
  constexpr int kWaves = kWM * kWN;
  constexpr int kMT = BM / (16 * kWM), kNT = BN / (16 * kWN);           // fragments of a wave
  constexpr int kXDma = BM / (8 * kWaves), kWDma = BN / (8 * kWaves);  // wave copies of 8 rows per stage
  constexpr int kDma = kXDma + kWDma;
  constexpr int kStageBytes = (BM + BN) * kTileK;
  static_assert(kXDma >= 1 && kWDma >= 1 && kStages >= 2 && (kStages - 1) * kDma <= 63, "tile does not fit the wave layout");
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / kWN, wn = wave % kWN;

  TileCursor tile, next;  // the tile being computed, and the one whose stages are being requested
  tile.at = next.at = blockIdx.x >> 3;
  tile.Place<BM, BN>(a, tiles);
  if (tile.rows == 0) return;
  next = tile;

  // Staging: copy i of a wave fills rows 8 (i kWaves + wave) .. + 7, lane l the 16 bytes at row l >> 3, place l & 7.  A row's
  // chunk c lies at place c ^ ((row >> 1) & 7): the 16 lanes whose reads the banks serve together - four rows of each
  // multiple of four, not all of the same chunk - then lie in 16 different 16-byte columns of the 256 bytes that the banks
  // span.
  static_assert(kWaves % 2 == 0, "a wave's rows share the parity of row >> 3");
  const int chunk = (lane & 7) ^ (lane >> 4) ^ ((wave & 1) * 4);
  unsigned x_off[kXDma], w_off[kWDma];
#pragma unroll
  for (int i = 0; i < kXDma; ++i)
    x_off[i] = static_cast<unsigned>((i * kWaves + wave) * 8 + (lane >> 3)) * static_cast<unsigned>(a.x_stride);
#pragma unroll
  for (int i = 0; i < kWDma; ++i)
    w_off[i] = static_cast<unsigned>((i * kWaves + wave) * 8 + (lane >> 3)) * static_cast<unsigned>(a.w_stride);
  const int stages = (a.k + kTileK - 1) / kTileK;  // of a tile
  __amdgpu_buffer_rsrc_t x_rsrc, w_rsrc;
  auto describe = [&]() {  // past the last tile: nothing, zeros arrive
    x_rsrc = Descriptor(a.x + next.m0 * a.x_stride, next.rows ? (next.rows - 1) * a.x_stride + a.k : 0);
    w_rsrc = Descriptor(a.w + next.n0 * a.w_stride, next.rows ? (next.columns - 1) * a.w_stride + a.k : 0);
  };
  describe();
  int issue_k = 0;   // k of the next stage to be requested
  int issue_at = 0;  // its place in the ring, bytes
  unsigned issue_off = 0;
  auto issue_begin = [&]() { issue_off = issue_k + chunk * 16 < a.k ? static_cast<unsigned>(issue_k + chunk * 16) : kOutside; };
  auto issue_one = [&](auto i) {
    constexpr int d = decltype(i)::value;
    if constexpr (d < kXDma) DmaToLds(x_rsrc, x_off[d] + issue_off, lds + issue_at + (d * kWaves + wave) * 1024);
    else DmaToLds(w_rsrc, w_off[d - kXDma] + issue_off, lds + issue_at + BM * kTileK + ((d - kXDma) * kWaves + wave) * 1024);
  };
  auto issue_end = [&]() {
    issue_at = issue_at + kStageBytes == kStages * kStageBytes ? 0 : issue_at + kStageBytes;
    issue_k += kTileK;
    if (issue_k >= a.k) {
      issue_k = 0;
      next.at += gridDim.x >> 3;
      next.Place<BM, BN>(a, tiles);
      describe();
    }
  };

  // Fragments: lane l holds row l & 15, k 64 h + 16 (l >> 4) .. + 15 for half h
  const int frag = (lane & 15) * kTileK + ((lane >> 4) ^ ((lane >> 1) & 7)) * 16;
  const int x_frag = wm * (BM / kWM) * kTileK + frag;
  const int w_frag = (BM + wn * (BN / kWN)) * kTileK + frag;
  int4v x[3][kMT], w[3][kNT];
  constexpr int kReads = kMT + kNT;  // of a half
  int read_at = 0;
  auto read_one = [&](auto half, auto set, auto i) {
    constexpr int h = decltype(half)::value, s = decltype(set)::value, d = decltype(i)::value;
    if constexpr (d < kNT) w[s][d] = *reinterpret_cast<const int4v*>(lds + ((read_at + w_frag) ^ (h * 64)) + d * 16 * kTileK);
    else x[s][d - kNT] = *reinterpret_cast<const int4v*>(lds + ((read_at + x_frag) ^ (h * 64)) + (d - kNT) * 16 * kTileK);
  };
  auto read_end = [&]() { read_at = read_at + kStageBytes == kStages * kStageBytes ? 0 : read_at + kStageBytes; };

  int4v acc[kMT][kNT];
  constexpr int kProducts = kMT * kNT;  // of a half
  // One stage; its halves are in sets 0 and `second`, the next stage's come to 0 and `third`.  A request or a read at most
  // between two products: a product occupies its unit for 16 cycles and the wave is free to issue for 12 of them; what does
  // not fit there leaves the unit idle.
  auto stage = [&](auto second, auto third) {
    constexpr int s = decltype(second)::value;
    issue_begin();
    Unrolled<0, kProducts>([&](auto t) {  // the place of this stage has been read by every wave: requested into
      constexpr int p = decltype(t)::value, i = p / kNT, j = p % kNT;
      Mfma(w[0][j], x[0][i], acc[i][j]);
      Unrolled<p * kDma / kProducts, (p + 1) * kDma / kProducts>(issue_one);
      __builtin_amdgcn_sched_barrier(0);
    });
    issue_end();
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * kDma) : "memory");  // the next stage is there
    __builtin_amdgcn_s_barrier();
    Unrolled<0, kProducts>([&](auto t) {
      constexpr int p = decltype(t)::value, i = p / kNT, j = p % kNT;
      Mfma(w[s][j], x[s][i], acc[i][j]);
      Unrolled<p * 2 * kReads / kProducts, (p + 1) * 2 * kReads / kProducts>([&](auto r) {
        constexpr int q = decltype(r)::value, h = q / kReads;
        if constexpr (h == 0) read_one(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{}, std::integral_constant<int, q>{});
        else read_one(std::integral_constant<int, 1>{}, third, std::integral_constant<int, q - kReads>{});
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    read_end();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and has been read
    __builtin_amdgcn_s_barrier();
  };

#pragma unroll
  for (int s = 0; s < kStages; ++s) {
    issue_begin();
    Unrolled<0, kDma>(issue_one);
    issue_end();
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * kDma) : "memory");
  __builtin_amdgcn_s_barrier();

  constexpr std::integral_constant<int, 0> kZero{};
  constexpr std::integral_constant<int, 1> kOne{};
  constexpr std::integral_constant<int, 2> kTwo{};
  while (true) {
    // The tile's first stage, here and not during the tile before: its registers serve that one's epilogue.
    Unrolled<0, kReads>([&](auto i) { read_one(kZero, kZero, i); });
    Unrolled<0, kReads>([&](auto i) { read_one(kOne, kOne, i); });
    read_end();
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        acc[i][j] = int4v{0, 0, 0, 0};
        Pin(acc[i][j]);
      }
    SettleAccumulators();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    for (int left = stages; left > 0; left -= 2) {
      stage(kOne, kTwo);
      if (left == 1) break;
      stage(kTwo, kOne);
    }
    read_at = read_at == 0 ? (kStages - 1) * kStageBytes : read_at - kStageBytes;  // what the last stage read is read again
    SettleAccumulators();
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
      for (int j = 0; j < kNT; ++j) Pin(acc[i][j]);
    int8_t* const mine = lds + kStages * kStageBytes + wave * (kNT * 1024);
    const int m = wm * (BM / kWM), n = wn * (BN / kWN);
    if (!a.vector_rows) FinishWave<T, kAny, true>(a, tile, m, n, mine, acc);
    else if (!a.line_rows) FinishWave<T, kPieces, true>(a, tile, m, n, mine, acc);
    else if (a.residual) FinishWave<T, kLines, true>(a, tile, m, n, mine, acc);
    else FinishWave<T, kLines, false>(a, tile, m, n, mine, acc);
    tile.at += gridDim.x >> 3;
    tile.Place<BM, BN>(a, tiles);
    if (tile.rows == 0) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing may arrive in this LDS after the block has left it
}

// Tiles for rows at any address, which the DMA does not take: a stage's pieces come to registers along the rows, as the
// DMA's lanes go, while the two stages before it are multiplied, and are written to the other half of LDS behind them.  Four
// waves.  Bound by those loads: of 16 bytes at odd addresses a CU takes in 14 to 17 bytes per cycle.  Between copying and
// the split kernels it has its place: 672 x 1308 x 133 5.1 us (copied 7.9, split 7.1), 200 x 4096 x 4095 22.6 (24.0, 26.1).
template <typename T, int BM, int BN, int kWM, int kWN, int kBlocks>
__global__ __launch_bounds__(256, kBlocks) void TileAnyKernel(LinearArgs a, Tiles tiles) {
  static_assert(kWM * kWN == 4, "four waves");
  constexpr int kMT = BM / (16 * kWM), kNT = BN / (16 * kWN);
  constexpr int kXPieces = BM / 32, kPieces = (BM + BN) / 32;
  constexpr int kStageBytes = (BM + BN) * kTileK;
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / kWN, wn = wave % kWN;
  TileCursor tile;
  tile.at = blockIdx.x >> 3;
  tile.Place<BM, BN>(a, tiles);
  if (tile.rows == 0) return;
  const int8_t* const x_rows = a.x + tile.m0 * a.x_stride;
  const int8_t* const w_rows = a.w + tile.n0 * a.w_stride;
  const int chunk = (lane & 7) ^ (lane >> 4) ^ ((wave & 1) * 4);  // the places in LDS as in TileKernel
  unsigned row[kPieces];  // offsets; rows past the end read the last one, their results are not stored
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    if (i < kXPieces) row[i] = min((i * 4 + wave) * 8 + (lane >> 3), tile.rows - 1) * static_cast<unsigned>(a.x_stride);
    else row[i] = min(((i - kXPieces) * 4 + wave) * 8 + (lane >> 3), tile.columns - 1) * static_cast<unsigned>(a.w_stride);
  }
  const int stages = (a.k + kTileK - 1) / kTileK;
  int4v piece[2][kPieces];  // of two stages, on their way
  auto load = [&](int s, auto set) {
    int4v (&to)[kPieces] = piece[decltype(set)::value];
    const int k = s * kTileK + chunk * 16;
    if (s * kTileK + kTileK <= a.k) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) __builtin_memcpy(&to[i], (i < kXPieces ? x_rows : w_rows) + (row[i] + k), 16);
    } else if (s < stages) {  // the rows end in this stage
#pragma unroll
      for (int i = 0; i < kPieces; ++i) to[i] = RequestPiece((i < kXPieces ? x_rows : w_rows) + row[i], k, a.k);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) to[i] = PieceOf(to[i], k, a.k);
    }
  };
  auto store = [&](int at, auto set) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      *reinterpret_cast<int4v*>(lds + at + (i * 4 + wave) * 1024 + lane * 16) = piece[decltype(set)::value][i];
  };
  const int frag = (lane & 15) * kTileK + ((lane >> 4) ^ ((lane >> 1) & 7)) * 16;
  const int x_frag = wm * (BM / kWM) * kTileK + frag;
  const int w_frag = (BM + wn * (BN / kWN)) * kTileK + frag;
  int4v acc[kMT][kNT];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) acc[i][j] = int4v{0, 0, 0, 0};
  constexpr std::integral_constant<int, 0> kZero{};
  constexpr std::integral_constant<int, 1> kOne{};
  // stage s from its half of LDS, whose pieces were of set `mine`: those of two stages on are requested into it, and the
  // other half, which every wave has read before the barrier behind the last stage, takes the next stage's
  auto stage = [&](int s, int at, auto mine, auto other) {
    load(s + 2, mine);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int4v x[kMT], w[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) w[j] = *reinterpret_cast<const int4v*>(lds + ((at + w_frag) ^ (h * 64)) + j * 16 * kTileK);
#pragma unroll
      for (int i = 0; i < kMT; ++i) x[i] = *reinterpret_cast<const int4v*>(lds + ((at + x_frag) ^ (h * 64)) + i * 16 * kTileK);
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x[i], acc[i][j], 0, 0, 0);
    }
    if (s + 1 < stages) store(kStageBytes - at, other);
    __syncthreads();
  };
  load(0, kZero);
  load(1, kOne);
  store(0, kZero);
  __syncthreads();
  for (int s = 0; s < stages; s += 2) {
    stage(s, 0, kZero, kOne);
    if (s + 1 < stages) stage(s + 1, kStageBytes, kOne, kZero);
  }
  int8_t* const mine = lds + wave * (kNT * 1024);
  const int m = wm * (BM / kWM), n = wn * (BN / kWN);
  if (!a.vector_rows) FinishWave<T, kAny, true>(a, tile, m, n, mine, acc);
  else FinishWave<T, kPieces, true>(a, tile, m, n, mine, acc);
}

// Rows that do not start at multiples of 16 bytes are copied to rows that do, zeros behind them: the DMA moves whole
// 16-byte pieces.  x's rows come first, w's behind them.  A thread has kPadPieces pieces on their way at a time.
constexpr int kPadPieces = 4;

__global__ __launch_bounds__(256) void PadKernel(LinearArgs a, int8_t* __restrict__ to, int pieces, int pitch) {
  const long long count = (a.m + a.n) * pieces;
  const long long first = static_cast<long long>(blockIdx.x) * (256 * kPadPieces) + threadIdx.x;
  int4v piece[kPadPieces];
  int8_t* at[kPadPieces];
  int k[kPadPieces];
#pragma unroll
  for (int j = 0; j < kPadPieces; ++j) {
    const long long i = min(first + j * 256, count - 1);  // the last one is written by several threads, with the same bytes
    const long long row = count >> 31 ? i / pieces : static_cast<unsigned>(i) / static_cast<unsigned>(pieces);
    k[j] = static_cast<int>(i - row * pieces) * 16;
    at[j] = to + row * pitch + k[j];
    piece[j] = RequestPiece(row < a.m ? a.x + row * a.x_stride : a.w + (row - a.m) * a.w_stride, k[j], a.k);
  }
#pragma unroll
  for (int j = 0; j < kPadPieces; ++j) *reinterpret_cast<int4v*>(at[j]) = PieceOf(piece[j], k[j], a.k);
}

int Status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : -1000 - static_cast<int>(e);
}

// More than 64 KB of LDS has to be allowed, once for each kernel and device.
template <auto* kKernel>
int AllowLds(int bytes) {
  static std::atomic<uint64_t> allowed{0};
  if (bytes <= 65536) return 0;
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  const uint64_t bit = 1ull << (device & 63);
  if (e == hipSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  return e == hipSuccess ? 0 : -1000 - static_cast<int>(e);
}

// A grid holds fewer than 2^32 threads: tokens beyond that go to further launches.
template <int BM, int BN, int kThreads, typename F>
int EachRun(const LinearArgs& a, F&& launch) {
  const long long tiles_n = (a.n + BN - 1) / BN;
  constexpr long long kMostBlocks = (1ll << 31) / kThreads;
  if (tiles_n > kMostBlocks) return -3;
  const long long most_m = kMostBlocks / tiles_n * BM;
  for (long long m = 0; m < a.m; m += most_m) {
    const long long left = a.m - m < most_m ? a.m - m : most_m;
    launch(static_cast<unsigned>((left + BM - 1) / BM * tiles_n), m, static_cast<unsigned>(tiles_n));
  }
  return Status();
}

template <int kMT, int kNT, int kWaves>
int LaunchSplitAny(const LinearArgs& a, hipStream_t stream) {
  constexpr int kLds = kWaves * (kMT + kNT) * 2048;
  static_assert((kMT + kNT) * 2 >= kMT * kNT, "the sums meet in the stages' place");
  if (const int rc = AllowLds<&SplitAnyKernel<kMT, kNT, kWaves>>(kLds)) return rc;
  return EachRun<16 * kMT, 16 * kNT, 64 * kWaves>(a, [&](unsigned blocks, long long m, unsigned tiles_n) {
    hipLaunchKernelGGL((SplitAnyKernel<kMT, kNT, kWaves>), dim3(blocks), dim3(64 * kWaves), kLds, stream, a, m, tiles_n);
  });
}

template <int kMT, int kNT, int kWaves, int kStages>
int LaunchSplitDma(const LinearArgs& a, hipStream_t stream) {
  constexpr int kLds = kWaves * kStages * (kMT + kNT) * 2048;
  static_assert(kLds <= 160 * 1024 && (kStages - 1) * 2 * (kMT + kNT) <= 63, "ring too large");
  if (const int rc = AllowLds<&SplitDmaKernel<kMT, kNT, kWaves, kStages>>(kLds)) return rc;
  return EachRun<16 * kMT, 16 * kNT, 64 * kWaves>(a, [&](unsigned blocks, long long m, unsigned tiles_n) {
    hipLaunchKernelGGL((SplitDmaKernel<kMT, kNT, kWaves, kStages>), dim3(blocks), dim3(64 * kWaves), kLds, stream, a, m, tiles_n);
  });
}

template <typename T, int BM, int BN, int kWM, int kWN, int kStages, int kBlocks>
int LaunchTile(const LinearArgs& a, hipStream_t stream) {
  const long long tiles_m = (a.m + BM - 1) / BM, tiles_n = (a.n + BN - 1) / BN;
  if (tiles_m * tiles_n > (1ll << 30)) return -3;
  const Tiles tiles{static_cast<unsigned>(tiles_m), static_cast<unsigned>(tiles_n), static_cast<unsigned>((tiles_m * tiles_n + 7) / 8)};
  constexpr int kLds = kStages * (BM + BN) * kTileK + 16 * BN * kWM * 4;
  static_assert(kBlocks * kLds <= 160 * 1024, "a CU's LDS");
  constexpr unsigned kPerXcd = 32 * kBlocks;  // blocks that an XCD's 32 CUs hold
  if (const int rc = AllowLds<&TileKernel<T, BM, BN, kWM, kWN, kStages, kBlocks>>(kLds)) return rc;
  hipLaunchKernelGGL((TileKernel<T, BM, BN, kWM, kWN, kStages, kBlocks>), dim3(8 * (tiles.run < kPerXcd ? tiles.run : kPerXcd)),
                     dim3(64 * kWM * kWN), kLds, stream, a, tiles);
  return Status();
}

constexpr long long kMostTiles = 1ll << 23;  // a grid of fewer than 2^32 threads

template <typename T, int BM, int BN, int kWM, int kWN, int kBlocks>
int LaunchTileAny(const LinearArgs& a, hipStream_t stream) {
  const long long tiles_m = (a.m + BM - 1) / BM, tiles_n = (a.n + BN - 1) / BN;
  if (tiles_m * tiles_n > kMostTiles) return -3;
  const Tiles tiles{static_cast<unsigned>(tiles_m), static_cast<unsigned>(tiles_n), static_cast<unsigned>((tiles_m * tiles_n + 7) / 8)};
  constexpr int kLds = 2 * (BM + BN) * kTileK;
  static_assert(kLds >= 16 * BN * kWM * 4 && kBlocks * kLds <= 160 * 1024, "a CU's LDS");
  if (const int rc = AllowLds<&TileAnyKernel<T, BM, BN, kWM, kWN, kBlocks>>(kLds)) return rc;
  hipLaunchKernelGGL((TileAnyKernel<T, BM, BN, kWM, kWN, kBlocks>), dim3(8 * tiles.run), dim3(256), kLds, stream, a, tiles);
  return Status();
}

bool Aligned(const void* x, const void* w, long long x_stride, long long w_stride, long long k) {
  return ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | x_stride | w_stride | k) & 15) == 0;
}

// A weight of at least half of the 256 MB behind the XCDs' caches has lost its beginning there when it is read again: 16 x
// 32768 x 4096 takes 24.8 instead of 27.8 us past them.  One of 64 MB that is read again at once takes 14.4 instead of 12.8.
constexpr long long kPassing = 128ll << 20;

// Descriptors hold 32-bit offsets: 256 rows of a tile have to stay below 2^30 bytes.
constexpr long long kMostStride = 1 << 20;

// Rows at whole lines: at other multiples of 16 every request of a line touches two (2048 x 4096 x 4096: 48.5 us with rows
// 16 bytes further apart than the lines, 40.4 at whole lines).
int PaddedRow(long long k) { return static_cast<int>((k + 127) / 128 * 128); }

// Which kernel takes a product: the one whose time comes out least.  A CU has `tiles` of them to work through, `blocks` at a
// time.  One alone needs step_alone for each 128 k (of each of `waves` parts of k) and end_alone besides; with all `blocks`
// of a CU at work, each of them takes its step and end from what they share.  Outputs at odd addresses lengthen the ends by
// `odd`.  In us, without the launch and apart from the time of the bytes from memory, which is the same for all.  Fitted to
// the times of 1700 products of random sizes (m to 8192, n and k to 16384; 550 for rows at any address): the choice is on
// average 1.9% behind the fastest kernel here, where "the largest tile that fills three quarters of the CUs" was 9% behind
// (6177 x 8769 x 128: 83 -> 54 us; 1985 x 1216 x 7488: 41 -> 32; 2213 x 6330 x 384: 30 -> 22).
struct Way {
  int rows, columns, waves, blocks;
  float step_alone, end_alone, step, end, odd;
};

float Estimate(const Way& w, long long m, long long n, long long k) {
  const long long tiles = (((m + w.rows - 1) / w.rows) * ((n + w.columns - 1) / w.columns) + 255) / 256;  // of a CU
  const float steps = static_cast<float>(((k + kStep - 1) / kStep + w.waves - 1) / w.waves);
  const float odd = n % 8 ? 1.f + w.odd : 1.f;
  const float alone = static_cast<float>((tiles + w.blocks - 1) / w.blocks) * (steps * w.step_alone + w.end_alone * odd);
  const float shared = static_cast<float>(tiles) * (steps * w.step + w.end * odd);
  return alone > shared ? alone : shared;
}

// Tiles at least half of whose rows would be empty are left out: few rows are bound by memory, where estimates meet.
template <int kCount>
int Fastest(const Way (&ways)[kCount], long long m, long long n, long long k, float* time = nullptr, int most_columns = 256,
            int count = kCount) {
  int best = -1;
  float least = 0.f;
  for (int i = 0; i < count; ++i) {
    if ((ways[i].rows > 16 && ways[i].rows >= 2 * m) || ways[i].columns > most_columns) continue;
    const float t = Estimate(ways[i], m, n, k);
    if (best < 0 || t < least) {
      best = i;
      least = t;
    }
  }
  if (time) *time = least;
  return best;
}

constexpr Way kAligned[] = {{256, 256, 1, 1, 1.16f, 6.96f, 0.18f, 0.80f, 0.86f}, {256, 128, 1, 1, 0.73f, 4.34f, 0.30f, 0.80f, 0.72f},
                            {128, 128, 1, 2, 0.39f, 2.78f, 0.46f, 1.43f, 0.60f}, {64, 128, 1, 2, 0.34f, 1.89f, 0.32f, 1.02f, 0.54f},
                            {64, 64, 1, 4, 0.26f, 1.50f, 0.20f, 0.62f, 0.39f},   {32, 64, 8, 1, 1.37f, 1.34f, 0.13f, 0.80f, 0.12f},
                            {32, 32, 4, 2, 0.31f, 1.37f, 0.42f, 0.90f, 0.26f},   {32, 16, 4, 3, 0.20f, 1.05f, 0.28f, 0.58f, 0.43f},
                            {16, 64, 8, 2, 0.84f, 1.03f, 0.96f, 0.68f, 0.38f},   {16, 32, 4, 3, 0.24f, 0.97f, 0.29f, 0.57f, 0.48f},
                            {16, 32, 2, 6, 0.23f, 0.90f, 0.16f, 0.37f, 0.50f},   {16, 16, 8, 2, 0.30f, 0.90f, 0.34f, 0.69f, 0.48f},
                            {16, 16, 4, 5, 0.20f, 0.76f, 0.18f, 0.40f, 0.62f},   {16, 16, 2, 10, 0.20f, 0.73f, 0.10f, 0.24f, 0.60f}};

// Few tokens are bound by memory, and what differs is how the rows that are asked for at a time fall on its channels, which
// the estimates do not know.  Tiles of 16 weight rows do best where rows are multiples of 8 KB apart: 16 x 6144 x 8192 13.5
// us, 15.5 with 32 rows; from 17 tokens on that is over (17 x 6144 x 8192: 14.6 with 16 rows, 14.8 with 64).  For up to eight
// tokens and a large weight one of them stands for all: 1 x 16384 x 8192 23.9 us (26.4 with 64 rows), 8 x 4096 x 16384
// 18.6 (25.4); with rows 4 KB apart 64 rows would do better (1 x 16384 x 4096 16.1 and not 16.9, 1 x 28672 x 4096 24.0 and
// not 27.2), and nine tokens, which the estimates place, have them (16.1 and 24.3).
constexpr long long kStreams = 64ll << 20;

int AlignedWay(const LinearArgs& a) {
  if (a.m <= 8 && a.n * a.k >= kStreams) return 12;
  return Fastest(kAligned, a.m, a.n, a.k, nullptr, a.m <= 16 && a.w_stride % 8192 == 0 ? 16 : 256);
}

template <typename T>
int LaunchAligned(int way, const LinearArgs& a, hipStream_t st) {
  switch (way) {
    case 0: return LaunchTile<T, 256, 256, 2, 2, 2, 1>(a, st);
    case 1: return LaunchTile<T, 256, 128, 2, 2, 3, 1>(a, st);
    case 2: return LaunchTile<T, 128, 128, 2, 2, 2, 2>(a, st);
    case 3: return LaunchTile<T, 64, 128, 2, 2, 2, 2>(a, st);
    case 4: return LaunchTile<T, 64, 64, 2, 2, 2, 4>(a, st);
    case 5: return LaunchSplitDma<2, 4, 8, 1>(a, st);
    case 6: return LaunchSplitDma<2, 2, 4, 2>(a, st);
    case 7: return LaunchSplitDma<2, 1, 4, 2>(a, st);
    case 8: return LaunchSplitDma<1, 4, 8, 1>(a, st);
    case 9: return LaunchSplitDma<1, 2, 4, 2>(a, st);
    case 10: return LaunchSplitDma<1, 2, 2, 2>(a, st);
    case 11: return LaunchSplitDma<1, 1, 8, 2>(a, st);
    case 12: return LaunchSplitDma<1, 1, 4, 2>(a, st);
    default: return LaunchSplitDma<1, 1, 2, 2>(a, st);
  }
}

constexpr Way kUnaligned[] = {{32, 64, 4, 3, 1.27f, 3.57f, 1.22f, 1.92f, 0.25f}, {32, 32, 8, 2, 1.71f, 1.25f, 1.50f, 0.69f, 0.38f},
                              {32, 32, 4, 4, 0.82f, 2.12f, 0.79f, 0.55f, 0.25f}, {16, 32, 4, 4, 0.60f, 1.58f, 0.59f, 0.40f, 0.33f},
                              {16, 16, 16, 1, 1.57f, 0.31f, 0.30f, 0.80f, 1.46f}, {16, 16, 4, 4, 0.45f, 1.10f, 0.41f, 0.11f, 0.46f},
                              {64, 64, 1, 4, 0.58f, 1.66f, 0.42f, 0.75f, 0.24f}};

bool FarApart(const LinearArgs& a) {
  return a.x_stride > kMostStride || a.w_stride > kMostStride || a.y_stride > kMostStride || a.residual_stride > kMostStride;
}

int UnalignedWay(const LinearArgs& a) {
  const bool tiles = !FarApart(a) && ((a.m + 63) / 64) * ((a.n + 63) / 64) <= kMostTiles;
  return Fastest(kUnaligned, a.m, a.n, a.k, nullptr, 256, tiles ? 7 : 6);
}

int LaunchUnaligned(int way, const LinearArgs& a, hipStream_t st) {
  switch (way) {
    case 0: return LaunchSplitAny<2, 4, 4>(a, st);
    case 1: return LaunchSplitAny<2, 2, 8>(a, st);
    case 2: return LaunchSplitAny<2, 2, 4>(a, st);
    case 3: return LaunchSplitAny<1, 2, 4>(a, st);
    case 4: return LaunchSplitAny<1, 1, 16>(a, st);
    case 5: return LaunchSplitAny<1, 1, 4>(a, st);
    default:
      if (a.dtype == tca::kF32) return LaunchTileAny<float, 64, 64, 2, 2, 4>(a, st);
      return a.dtype == tca::kF16 ? LaunchTileAny<_Float16, 64, 64, 2, 2, 4>(a, st) : LaunchTileAny<Bf16, 64, 64, 2, 2, 4>(a, st);
  }
}

// Copying the operands to aligned rows lets the DMA and the large tiles in; it costs a launch and the operands' bytes twice
// (3.5 us and 0.4 us per MB).  1756 x 1856 x 4199: 29 us copied, 88 as they are; 125 x 5248 x 2315: 19.2 and 16.4.
bool Pads(long long m, long long n, long long k) {
  float aligned, unaligned;
  Fastest(kAligned, m, n, k, &aligned);
  Fastest(kUnaligned, m, n, k, &unaligned);
  return aligned + 3.5f + 4.0e-7f * static_cast<float>(m + n) * static_cast<float>(k) < unaligned;
}

// How a product is computed: the entry of kAligned or, less `any`, of kUnaligned, and whether its operands are copied first.
struct Choice {
  bool copied, any;
  int way;
};

// `a` becomes what the kernel is called with: where the operands are copied, rows of the workspace.
Choice Choose(LinearArgs& a, void* workspace) {
  Choice c{};
  if (!Aligned(a.x, a.w, a.x_stride, a.w_stride, a.k)) {
    c.copied = Pads(a.m, a.n, a.k);
    c.any = !c.copied;
    if (c.copied) {
      const int row = PaddedRow(a.k);
      a.x = static_cast<const int8_t*>(workspace);
      a.w = workspace ? a.x + a.m * row : nullptr;
      a.x_stride = a.w_stride = row;
      a.k = (a.k + 15) / 16 * 16;
    }
  }
  c.any = c.any || FarApart(a);
  c.way = c.any ? UnalignedWay(a) : AlignedWay(a);
  return c;
}

int Launch(const LinearArgs& given, void* workspace, hipStream_t st) {
  LinearArgs a = given;
  const Choice c = Choose(a, workspace);
  if (c.copied) {
    if (!workspace) return -4;
    const int pieces = a.k / 16;
    const long long blocks = ((a.m + a.n) * pieces + 256 * kPadPieces - 1) / (256 * kPadPieces);
    if (blocks >= 1 << 24) return -3;
    hipLaunchKernelGGL(PadKernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, given, static_cast<int8_t*>(workspace), pieces,
                       static_cast<int>(a.x_stride));
  }
  if (c.any) return LaunchUnaligned(c.way, a, st);
  if (a.dtype == tca::kF32) return LaunchAligned<float>(c.way, a, st);
  return a.dtype == tca::kF16 ? LaunchAligned<_Float16>(c.way, a, st) : LaunchAligned<Bf16>(c.way, a, st);
}

}  // namespace

extern "C" {

// Bytes of workspace (at a multiple of 16) that a launch with these operands needs; mostly 0.
long long tca_int8_linear_workspace_bytes(const void* x, const void* w, long long m, long long n, long long k, long long x_stride,
                                          long long w_stride) {
  if (m <= 0 || n <= 0 || k <= 0 || Aligned(x, w, x_stride, w_stride, k) || !Pads(m, n, k)) return 0;
  return (m + n) * PaddedRow(k);
}

// Which kernel takes a product of these operands: 0 to 13 the tiles for aligned rows, 16 to 22 those for rows at any address;
// 32 more where the operands are copied to aligned rows first.  -1 for operands that a launch refuses.
int tca_int8_linear_way(const void* x, const void* w, long long m, long long n, long long k, long long x_stride, long long w_stride,
                        long long residual_stride, long long y_stride) {
  if (m <= 0 || n <= 0 || k <= 0 || k > 131071) return -1;
  LinearArgs a{};
  a.x = static_cast<const int8_t*>(x);
  a.w = static_cast<const int8_t*>(w);
  a.m = m;
  a.n = n;
  a.k = static_cast<int>(k);
  a.x_stride = x_stride;
  a.w_stride = w_stride;
  a.residual_stride = residual_stride;
  a.y_stride = y_stride;
  const Choice c = Choose(a, nullptr);
  return (c.copied ? 32 : 0) + (c.any ? 16 : 0) + c.way;
}

int tca_int8_linear_launch(const void* x, const void* x_scale, const void* w, const void* w_scale, const void* bias,
                           const void* residual, void* y, int dtype, long long m, long long n, long long k,
                           long long x_stride, long long w_stride, long long residual_stride, long long y_stride,
                           void* workspace, void* stream) {
  if (!x || !x_scale || !w || !w_scale || !y || m <= 0 || n <= 0 || k <= 0) return -1;
  if (dtype != tca::kF32 && dtype != tca::kF16 && dtype != tca::kBF16) return -2;
  if (k > 131071 || (reinterpret_cast<uintptr_t>(workspace) & 15)) return -3;
  const int size = dtype == tca::kF32 ? 4 : 2;
  const bool vector_rows = ((reinterpret_cast<uintptr_t>(w_scale) | reinterpret_cast<uintptr_t>(bias) |
                             reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual) |
                             static_cast<uintptr_t>((n | y_stride | (residual ? residual_stride : 0)) * size)) & 15) == 0;
  const bool line_rows = ((reinterpret_cast<uintptr_t>(y) | static_cast<uintptr_t>(y_stride * size)) & 127) == 0;
  const LinearArgs a{static_cast<const int8_t*>(x), static_cast<const float*>(x_scale), static_cast<const int8_t*>(w),
                     static_cast<const float*>(w_scale), bias, residual, y, m, n, x_stride, w_stride,
                     residual ? residual_stride : 0, y_stride, static_cast<int>(k), dtype,
                     m <= 16 && n * k >= kPassing, vector_rows, line_rows};
  return Launch(a, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
