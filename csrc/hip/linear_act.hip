// Matrix products of dense layers, with bias, activation and residual in the
// epilogue, and their gradients.
//
//   z = x W^T + b      y = act(z) + r
//   dz = dy act'(z)    dx = dz W           dW = dz^T x      db = sum dz
//
// What is kept for the backward: act'(z), formed where z is still in fp32, so
// that no erf or exp is computed twice. With 16-bit tensors it has 16 bits too:
// from 2^-7 on (2^-6 for fp16) steps of 2^-15, where bf16's or fp16's own
// rounding would show in dx and dW, and below that 8 (9) bits of mantissa down
// to 2^-52 (2^-28): fixed point alone would lose the small derivatives of GELU
// below -4 and SiLU below -9 in part, and below -4.84 and -13.6 in whole. A
// kept one is off by 2^-16 at most, and below those borders by 2^-9 (2^-10) of
// itself, half of bf16's own rounding. ReLU's 0 and 1 are exact.
//
// dz of 16-bit tensors has more bits than they do, where act'(z) is no 0 or 1.
// The matrix cores take it as two numbers, the nearest one and what that has
// lost (db sums it as it is): with one alone dx and dW were off by sqrt(2) of
// their own rounding, and by 2 to 3 times that where their terms cancel. Each
// step of k is then two, one for either part, the other operand the same, which
// comes from the L2: 1024x1024 from 3999 in fp16 29 us in place of 17 (dW) and
// 22 of 15 (dx), 8192x4096x4096 bf16 with all gradients 1060 in place of 668.
//
// All three products are one kernel, D[m][n] = sum_k X(m,k) Y(n,k), where
// either operand may lie with k consecutive or with its own index
// consecutive:
//   forward X = x, Y = W;  dx: X = dz, Y = W (n consecutive);
//   dW: X = dz, Y = x (both with their own index consecutive).
//
// A workgroup computes a kBM x kBN tile, waves in a grid over it. Each step
// takes 128 bytes of k from both operands through LDS, from memory directly,
// 16 bytes a lane, kAhead steps ahead: kAhead + 1 buffers of X and kAhead of
// Y, since X's next loads go where the last step's were and Y's where this
// step's first half was. The next half step's fragments are read from LDS
// during this half's products. The bounds are the buffer descriptor's: rows
// and columns past the end read as 0. Lanes of one load go to consecutive LDS
// addresses, so what would be a column of equal banks is spread by choosing
// which 16 bytes a lane fetches (an exclusive or with the row's bits).
// Operands with k consecutive are read from LDS 16 bytes a lane; with 16-bit
// types the others go through the transposing LDS read, 4 values of k a
// lane. Y is the matrix instruction's row operand, so that a lane ends up
// with 4 consecutive columns of one row of D.
//
// Few tiles: the k axis is split, partial sums go to memory in fp32 and a
// second kernel adds them in order and applies the epilogue.
//
// What bounds it, measured on one MI355X in bf16 (times of a kernel):
//   256-wide tiles: the matrix cores and the card's power. 32000x12544x1024
//     with bias and ReLU 620 us, 1330 TFLOP/s; products without any load
//     reach 1450 to 1530 on such data, the library's product alone 1250. The
//     matrix cores are busy 73% of the cycles, LDS has no bank conflicts.
//     Four waves of 512 registers were slower than eight of 256.
//   128-wide tiles: LDS. In a step waves with 64x64 of it read 64 KB (those
//     with 64x32 96 KB) and the loads write 32 KB, 768 cycles (1024) at 128
//     bytes each, for 515 cycles of products: 0.48 us (0.55), 1120 TFLOP/s.
//     1000x12544x1024 in 4 splits 31 us and 5 to add them up; the library 45.
//   64-wide tiles: with many steps the L2s, which give 20 TB/s (dW of
//     3999x1024x1024 17 us); with few the latency of loads and of the launch:
//     100x1024x81 7.2 us, of which a launch of one step takes 5.
//   fp32: the matrix cores, busy 94% at 4096x4096x4096: 145 TFLOP/s forward and
//     backward (the library's 8192x8192x8192 153), 104 to 119 at 3999x1024x1024.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "train_ops.h"
#include "typed.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef fp16_t fp16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kRow = 128;                 // bytes of k in one step
constexpr unsigned kOutside = 0x80000000u;  // above any descriptor's range

// One packet of 16 bytes an operand; the products of all its values.
__device__ inline void mma(f32x4& acc, i32x4 a, i32x4 b, bf16_t) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0,
      0);
}
__device__ inline void mma(f32x4& acc, i32x4 a, i32x4 b, fp16_t) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), acc, 0, 0,
      0);
}
__device__ inline void mma(f32x4& acc, i32x4 a, i32x4 b, float) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(a[j]),
                                               __int_as_float(b[j]), acc, 0,
                                               0, 0);
}

// 16 bytes a lane from memory to LDS at `to` + 16 * lane. In assembly, as
// the compiler would wait for it before every transposing LDS read; there is
// no output register, and the waits are the caller's.
__device__ inline void load_lds(i32x4 desc, unsigned from, unsigned to) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(to), "v"(from), "s"(desc)
      : "memory", "m0");
}

// All but the latest kLater loads into LDS have arrived and every read of it
// is done, in all waves.
template <int kLater>
__device__ inline void arrived() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLater)
               : "memory");
}

__device__ inline i32x4 descriptor(const char* base, int bytes) {
  const unsigned long a = (unsigned long)base;
  i32x4 d;
  d[0] = __builtin_amdgcn_readfirstlane((int)a);
  d[1] = __builtin_amdgcn_readfirstlane((int)(a >> 32) & 0xffff);
  d[2] = bytes;
  d[3] = 0x00020000;
  return d;
}

// Bytes that a step may read of an operand with k consecutive: to the end of
// the last row's part in it, `left` packets from the row's end. A row of
// fewer than 128 bytes ends the range earlier, or the rows behind the last
// one would begin inside it. (A row is never longer than `ld`, so they are
// outside.)
constexpr __host__ __device__ int step_range(int rows, int ld, int left) {
  return (rows - 1) * ld + (left < 0 ? 0 : left * 16 < kRow ? left * 16 : kRow);
}
static_assert(step_range(3, 16, 1) == 48 && step_range(1, 16, 1) == 16,
              "rows of 16 bytes end with their own");
static_assert(step_range(2, 4096, 8) == 4096 + 128 &&
                  step_range(2, 4096, 200) == 4096 + 128,
              "a whole step of long rows");
static_assert(step_range(2, 176, 3) == 176 + 48, "the last step of rows");

// One operand's tile of kR rows (its own index) and 128 bytes of k.
template <typename T, bool kTrans, int kR, int kWaves>
struct Operand {
  static constexpr int kPer = 16 / sizeof(T);           // values of a packet
  static constexpr int kK = kRow / sizeof(T);           // k of one step
  static constexpr int kBytes = kR * kRow;
  static constexpr int kLoads = kBytes / (1024 * kWaves);
  static_assert(kLoads * 1024 * kWaves == kBytes, "whole loads for each wave");
  // With its own index consecutive: packets of one row of k, and how many
  // packets the 16 indices of a matrix operand take.
  static constexpr int kPackets = kR / kPer;
  static constexpr int kUnit = 16 / kPer;
  static constexpr int kUnits = kPackets / kUnit;

  const char* base;     // at the tile's first row, k = 0
  long second;          // from there to the second part
  int ld;               // bytes
  int rows;             // of this tile
  int k;                // k altogether
  unsigned from[kLoads];
  int packet[2];        // k consecutive: the packet that a lane fetches in
                        // even and odd loads
  static_assert(kLoads % 2 == 0, "even loads for each wave");

  static __device__ int twist(int r) {
    if constexpr (!kTrans) return (r >> 1) & 7;
    // The rows of k that one read takes fall on different banks: 8 g + 0..3
    // for 16-bit types, two g at a time, 4 g for fp32. Rows of 128 bytes lie
    // on the two halves of the banks in turn, which is the lowest bit.
    const int g = (r >> 3) & 1;
    const int f = sizeof(T) == 4 ? (r >> 2) & 3
                  : kUnits == 4  ? ((r >> 1) & 1) | g << 1
                                 : (r & 3) | g << 2;
    static_assert(kUnits == 4 || kUnits >= 8, "f is below the units");
    return f;
  }

  __device__ void init(const void* p, long ld_values, int first, int total,
                       int k_total, int wave, int lane, long to_second) {
    second = to_second;
    ld = (int)(ld_values * (long)sizeof(T));
    k = k_total;
    rows = total - first < kR ? total - first : kR;
    base = (const char*)p + (kTrans ? first * (long)sizeof(T)
                                    : first * (long)ld);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = (wave * kLoads + i) * 64 + lane;    // packet in LDS
      if constexpr (!kTrans) {
        const int r = at >> 3, c = (at & 7) ^ twist(r);
        from[i] = (unsigned)(r * ld + c * 16);
        packet[i & 1] = c;
      } else {
        const int r = at / kPackets, s = at % kPackets;
        const int c = ((s / kUnit) ^ twist(r)) * kUnit + s % kUnit;
        from[i] = (unsigned)(r * ld + c * 16);
      }
    }
  }

  struct Step {
    i32x4 desc;
    int left;           // k consecutive: packets left in the rows
  };

  // Step `step`'s part of the operand; from `end` on nothing is in range.
  // kTwo: steps go in pairs of the same k, the odd ones in the second part.
  template <bool kTwo>
  __device__ Step at_step(int step, int end) const {
    const int at = kTwo ? step >> 1 : step;
    const int k0 = at * kK, left = step < end ? k - k0 : 0;
    const char* part = kTwo && step & 1 ? base + second : base;
    if constexpr (!kTrans)
      return {descriptor(part + (long)at * kRow,
                         step_range(rows, ld, left / kPer)),
              left / kPer};
    const int rows_k = left < kK ? left : kK;
    return {descriptor(part + (long)k0 * ld,
                       rows_k > 0 ? (rows_k - 1) * ld + rows * (int)sizeof(T)
                                  : 0),
            0};
  }

  // Load i of the step; `to`: LDS address of the tile. In the last step of
  // a ragged k the packets past it would be the next row's.
  __device__ void load(const Step& s, int i, unsigned to, int wave) const {
    const unsigned f = kTrans || packet[i & 1] < s.left ? from[i] : kOutside;
    load_lds(s.desc, f, to + (wave * kLoads + i) * 1024);
  }

  // The packet of rows r0 + lane % 16 and k-group lane / 16 of half `h`.
  static __device__ i32x4 read(const char* tile, int r0, int h, int lane) {
    const int g = (lane >> 4) + 4 * h, i = lane & 15;
    if constexpr (!kTrans) {
      const int r = r0 + i;
      return *(const i32x4*)(tile + r * kRow + ((g ^ twist(r)) << 4));
    } else if constexpr (sizeof(T) == 2) {
      i32x4 out;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = g * 8 + q * 4 + (i >> 2);
        const char* p = tile + r * (kR * 2) +
                        (((r0 >> 4) ^ twist(r)) << 5) + ((i & 3) << 3);
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)p);
        const long two = __builtin_bit_cast(long, v);
        out[2 * q] = (int)two;
        out[2 * q + 1] = (int)(two >> 32);
      }
      return out;
    } else {
      i32x4 out;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = g * 4 + j;
        out[j] = *(const int*)(tile + r * (kR * 4) +
                               (((r0 >> 4) ^ twist(r)) << 6) + (i << 2));
      }
      return out;
    }
  }
};

// ---------------------------------------------------------------- epilogue

// The normal distribution at z: its density's exponential and its integral.
// fp32 tensors take erfc, whose small values below 0 do not cancel as 1 + erf
// does; for 16-bit ones the integral is Abramowitz and Stegun's 7.1.26, off by
// 7.5e-8 at most and a fifth of erf's instructions, which took 10 us of a 25 us
// forward of 3999x1024x1024. The exponential's instruction, and below the
// reciprocal's, are for 16 bits likewise: with the factor's rounding they are
// off by 0.5 |z| units in fp32's last place, 40 at the far end of SiLU.
template <typename T>
__device__ inline float exponential(float x) {
  return sizeof(T) == 4 ? expf(x) : __expf(x);
}

template <typename T>
__device__ inline void normal(float z, float& e, float& cdf) {
  e = exponential<T>(-0.5f * z * z);
  if constexpr (sizeof(T) == 4) {
    cdf = 0.5f * erfcf(z * -0.70710678f);
  } else {
    const float t =
        __builtin_amdgcn_rcpf(1.0f + 0.3275911f * 0.70710678f * fabsf(z));
    const float p =
        t * (0.254829592f +
             t * (-0.284496736f +
                  t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    const float tail = 0.5f * p * e;
    cdf = z < 0.0f ? tail : 1.0f - tail;
  }
}

template <typename T>
__device__ inline float sigmoid(float z) {
  const float d = 1.0f + exponential<T>(-z);
  return sizeof(T) == 4 ? 1.0f / d : __builtin_amdgcn_rcpf(d);
}

// act(z); slope: act'(z), of the same exponential.
template <typename T, int kAct>
__device__ inline float activate(float z, float& slope) {
  if constexpr (kAct == kActRelu) {
    slope = z > 0.0f ? 1.0f : 0.0f;
    return z < 0.0f ? 0.0f : z;                             // NaN stays
  }
  if constexpr (kAct == kActSilu) {
    const float s = sigmoid<T>(z);
    slope = s * (1.0f + z * (1.0f - s));
    return z * s;
  }
  if constexpr (kAct == kActGelu) {
    float e, cdf;
    normal<T>(z, e, cdf);
    slope = cdf + z * (0.39894228f * e);
    return z * cdf;
  }
  slope = 1.0f;
  return z;
}

// The derivative as it is kept: fp32 as it is; else a code of its magnitude in
// 14 bits, or 16 where it is above zero (all derivatives lie between -0.13 and
// 1.13): the two highest bits together are the sign, the last code is NaN.
// Magnitudes from `line` on are whole numbers of 2^-15. Those below are the
// exponent and first `bits` bits of an fp32 number times a power of two, which
// makes the codes meet at `line` and the smallest ones subnormal. bf16 has dz's
// exponents to go with 2^-52; in fp16 dz ends at 2^-24 and has more bits.
template <typename T>
using Kept = std::conditional_t<sizeof(T) == 4, float, unsigned short>;

template <typename T>
struct Code16 {
  static constexpr int bits = std::is_same_v<T, fp16_t> ? 9 : 8;
  static constexpr int below = 11776;               // codes below the line
  static constexpr int drop = 23 - bits;            // bits of fp32's mantissa
  static constexpr float line = 1.0f / (1 << (15 - bits));
  // Whole numbers of 2^-15 start at 2^bits on the line.
  static constexpr int shift = below - (1 << bits);
  // The line's exponent is 127 + bits - 15, its code's below >> bits.
  static constexpr int scale = 127 + bits - 15 - (below >> bits);
  static_assert(below % (1 << bits) == 0 && scale > 0, "whole binades");
  static_assert(shift + 36993 < 0xc000 && shift + 4225 < 0x3fff,
                "GELU's 1.1289 and -0.1289 have codes");
};

template <typename T>
__device__ inline Kept<T> keep(float slope) {
  if constexpr (sizeof(T) == 4) {
    return slope;
  } else {
    using C = Code16<T>;
    const float a = fabsf(slope);
    const unsigned b =
        __float_as_uint(a * __int_as_float((127 - C::scale) << 23));
    const unsigned few =
        (b + (1 << (C::drop - 1)) - 1 + ((b >> C::drop) & 1)) >> C::drop;
    const unsigned whole = (unsigned)(int)rintf(a * 32768.0f) + C::shift;
    const unsigned code =
        (a < C::line ? few : whole) | (slope < 0.0f ? 0xc000u : 0u);
    return (Kept<T>)(slope == slope ? code : 0xffffu);
  }
}

template <typename T>
__device__ inline float kept(Kept<T> k) {
  if constexpr (sizeof(T) == 4) {
    return k;
  } else {
    using C = Code16<T>;
    const bool negative = k >= 0xc000;
    const unsigned code = negative ? k & 0x3fffu : k;
    const float few = __uint_as_float(code << C::drop) *
                      __int_as_float((127 + C::scale) << 23);
    const float whole = (float)((int)code - C::shift) * (1.0f / 32768.0f);
    const float a = code < C::below ? few : whole;
    return k == 0xffff ? __int_as_float(0x7fc00000) : negative ? -a : a;
  }
}

constexpr int kOut = 8;       // consecutive columns that a lane finishes

// The bias of columns n .. n + 7, zeros past N.
template <typename T>
__device__ inline void load_bias(const LinearEpilogue& e, int n, int N,
                                 float (&b)[kOut]) {
#pragma unroll
  for (int i = 0; i < kOut; ++i)
    b[i] = e.bias != nullptr && n + i < N ? (float)((const T*)e.bias)[n + i]
                                          : 0.0f;
}

// 8 columns of a row as they lie in memory.
template <typename T>
struct Raw {
  i32x4 q[sizeof(T) * kOut / 16];
};

// The residual's columns n .. n + 7 of row m, if all are there.
template <typename T>
__device__ inline Raw<T> load_residual(const LinearEpilogue& e, long m, int n,
                                       int N) {
  Raw<T> r = {};
  if (e.residual != nullptr && n + kOut <= N)
    __builtin_memcpy(&r, (const T*)e.residual + m * e.ld_residual + n,
                     sizeof(r));
  return r;
}

// Columns n .. n + 7 of row m; `raw` is load_residual()'s.
template <typename T, int kAct>
__device__ inline void finish(const LinearEpilogue& e, long m, int n, int N,
                              const float (&b)[kOut], Raw<T> raw,
                              float (&z)[kOut]) {
  T* out = (T*)e.y + m * (long)N + n;
  using K = Kept<T>;
  K* slopes = e.kept ? (K*)e.kept + m * (long)N + n : nullptr;
  float slope;
  if (kAct != kActNone && slopes) {
    K k[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
      z[i] = activate<T, kAct>(z[i] + b[i], slope);
      k[i] = keep<T>(slope);
    }
    if (n + kOut <= N) {
      __builtin_memcpy(slopes, k, sizeof(k));
    } else {
#pragma unroll
      for (int i = 0; i < kOut; ++i)
        if (n + i < N) slopes[i] = k[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kOut; ++i)
      z[i] = activate<T, kAct>(z[i] + b[i], slope);
  }
  if (n + kOut <= N) {
    typedef T Res __attribute__((ext_vector_type(kOut)));
    const Res r = __builtin_bit_cast(Res, raw);
#pragma unroll
    for (int i = 0; i < kOut; ++i) z[i] += (float)r[i];
    store_f32<T, kOut>(out, z);
    return;
  }
  const T* res = (const T*)e.residual + m * e.ld_residual + n;
#pragma unroll
  for (int i = 0; i < kOut; ++i)
    if (n + i < N)
      out[i] = (T)(z[i] + (e.residual ? (float)res[i] : 0.0f));
}

// f(the activation as a constant)
template <typename F>
__device__ inline void with_act(int act, F f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    default: f(std::integral_constant<int, kActNone>{});
  }
}

// ------------------------------------------------------------------ kernel

// kWM x kWN waves over the tile, in kGroups that each take a part of the
// steps, with buffers of their own. Two waves a SIMD have 256 registers each,
// which holds the sums in ordinary ones: with more, the compiler moves
// hundreds of sums between the two kinds in each step.
template <typename T, bool kXT, bool kYT, bool kTwo, int kBM, int kBN, int kWM,
          int kWN, int kGroups, int kAhead>
__global__ __launch_bounds__(kWM * kWN * kGroups * 64, 2) void product_kernel(
    LinearProduct a) {
  constexpr int kWaves = kWM * kWN;
  using X = Operand<T, kXT, kBM, kWaves>;
  using Y = Operand<T, kYT, kBN, kWaves>;
  constexpr int kMI = kBM / kWM / 16, kNI = kBN / kWN / 16;
  constexpr int kYAt = (kAhead + 1) * X::kBytes;
  constexpr int kLds = kYAt + kAhead * Y::kBytes;
  __shared__ __attribute__((aligned(1024))) char lds_all[kGroups * kLds];

  // Workgroups go round the 8 chiplets; each gets a consecutive run of tiles,
  // blocks of `group` rows of tiles by all columns, down the rows first, so
  // that what runs at a time shares rows of X and of Y in the chiplet's L2.
  const int tiles_n = (a.n + kBN - 1) / kBN, tiles_m = (a.m + kBM - 1) / kBM;
  const int total = gridDim.x, xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
  const int big = total >> 3, rest = total & 7;
  const int id = xcd * big + (xcd < rest ? xcd : rest) + at;
  const int split = id / (tiles_m * tiles_n), tile = id % (tiles_m * tiles_n);
  const int block = tile / (a.group * tiles_n), in = tile % (a.group * tiles_n);
  const int deep = tiles_m - block * a.group < a.group
                       ? tiles_m - block * a.group : a.group;
  const int m0 = (block * a.group + in % deep) * kBM, n0 = in / deep * kBN;

  const int lane = threadIdx.x & 63;
  const int id_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = id_wave / kWaves, wave = id_wave % kWaves;
  char* lds = lds_all + group * kLds;
  const int xr = wave / kWN * (kBM / kWM), yr = wave % kWN * (kBN / kWN);
  X x;
  Y y;
  x.init(a.x, a.ldx, m0, a.ext_x, a.kx, wave, lane, a.second);
  y.init(a.y, a.ldy, n0, a.ext_y, a.ky, wave, lane, 0);

  const int steps = (a.kx + X::kK - 1) / X::kK * (kTwo ? 2 : 1);
  const int first_all = split * a.steps_per_split;
  const int last_all = first_all + a.steps_per_split < steps
                           ? first_all + a.steps_per_split : steps;
  // All groups take as many turns, the last ones perhaps past their steps,
  // where they get zeros.
  const int turns = (last_all - first_all + kGroups - 1) / kGroups;
  const int first = first_all + group * turns;
  const int last = first + turns < last_all ? first + turns : last_all;
  const unsigned at_lds =
      (unsigned)(unsigned long)(lds_char*)&lds_all[0] + group * kLds;

  f32x4 acc[kMI][kNI] = {};
  i32x4 xf[2][kMI], yf[2][kNI];
  const auto load_x = [&](int step, unsigned to) {
    const auto s = x.template at_step<kTwo>(step, last);
#pragma unroll
    for (int i = 0; i < X::kLoads; ++i) x.load(s, i, at_lds + to, wave);
  };
  const auto load_y = [&](int step, unsigned to) {
    const auto s = y.template at_step<kTwo>(step, last);
#pragma unroll
    for (int i = 0; i < Y::kLoads; ++i) y.load(s, i, at_lds + to, wave);
  };
  // Fragment r of a half step: one of X, all of Y, the rest of X, the order
  // in which the products need them.
  const auto read = [&](int r, int h, int xat, int yat) {
    if (r >= 1 && r <= kNI)
      yf[h][r - 1] = Y::read(lds + yat, yr + (r - 1) * 16, h, lane);
    else if (r < kMI + kNI)
      xf[h][r ? r - kNI : 0] =
          X::read(lds + xat, xr + (r ? r - kNI : 0) * 16, h, lane);
  };

  // Loads are kAhead steps ahead, of X in a step's first half into the buffer
  // of the step before, of Y in its second into this step's own, which all
  // waves have left by then.
#pragma unroll
  for (int d = 0; d < kAhead; ++d) {
    load_x(first + d, d * X::kBytes);
    load_y(first + d, kYAt + d * Y::kBytes);
  }
  int x0 = 0, x1 = X::kBytes, xw = kAhead * X::kBytes;
  int y0 = kYAt, y1 = kYAt + (kAhead > 1 ? Y::kBytes : 0);
  arrived<(kAhead - 1) * (X::kLoads + Y::kLoads)>();
#pragma unroll
  for (int r = 0; r < kMI + kNI; ++r) read(r, 0, x0, y0);
  // A half step: its products, row of fragments by row; the reads of the next
  // half's fragments, all but the last rows' time ahead of their use; and
  // loads of a later step, spread evenly, as four at a time on a CU's four
  // SIMDs would queue. The barrier is in the middle of the step: behind it
  // the next step has arrived and no wave still reads this one.
  constexpr int kReads = (kMI + kNI + kMI - 1) / kMI < 2
                             ? 2 : (kMI + kNI + kMI - 1) / kMI;
  for (int s = first; s < first + turns; ++s) {
    const auto xs = x.template at_step<kTwo>(s + kAhead, last);
#pragma unroll
    for (int i = 0; i < kMI; ++i) {
#pragma unroll
      for (int l = i * X::kLoads / kMI; l < (i + 1) * X::kLoads / kMI; ++l)
        x.load(xs, l, at_lds + xw, wave);
#pragma unroll
      for (int r = i * kReads; r < (i + 1) * kReads; ++r) read(r, 1, x0, y0);
#pragma unroll
      for (int j = 0; j < kNI; ++j) mma(acc[i][j], yf[0][j], xf[0][i], T{});
      __builtin_amdgcn_sched_barrier(0);
    }
    arrived<(kAhead - 1) * X::kLoads + (kAhead - 2) * Y::kLoads>();
    const auto ys = y.template at_step<kTwo>(s + kAhead, last);
#pragma unroll
    for (int i = 0; i < kMI; ++i) {
#pragma unroll
      for (int l = i * Y::kLoads / kMI; l < (i + 1) * Y::kLoads / kMI; ++l)
        y.load(ys, l, at_lds + y0, wave);
#pragma unroll
      for (int r = i * kReads; r < (i + 1) * kReads; ++r) read(r, 0, x1, y1);
#pragma unroll
      for (int j = 0; j < kNI; ++j) mma(acc[i][j], yf[1][j], xf[1][i], T{});
      __builtin_amdgcn_sched_barrier(0);
    }
    xw = x0, x0 = x1, y0 = y1;
    x1 = x1 + X::kBytes == kYAt ? 0 : x1 + X::kBytes;
    y1 = y1 + Y::kBytes == kLds ? kYAt : y1 + Y::kBytes;
  }

  // A lane holds row lane % 16 and columns 4 (lane / 16) .. + 3 of each
  // 16 x 16 part. The parts go through the wave's share of LDS (packets of a
  // row in an order that spreads the banks), from where a lane takes 8
  // consecutive columns: full-width accesses, and one copy of the epilogue's
  // code.
  constexpr int kCols = kBN / kWN, kQuads = kCols / 4;
  constexpr int kOwn = kMI / kGroups;        // parts down that a group finishes
  constexpr int kSums = kGroups > 1 ? kWaves * kOwn * kNI * 64 * 16 : 0;
  constexpr int kFit = (kLds - kSums) / kWaves / (16 * kCols * 4);
  constexpr int kParts = kFit >= kOwn ? kOwn : kFit >= kOwn / 2 ? kOwn / 2
                                                                : kOwn / 4;
  static_assert(kParts > 0 && kParts <= kFit, "a wave's share of LDS");
  constexpr int kLanes = kCols / kOut;                     // of one row
  arrived<0>();
  if constexpr (kGroups > 1) {
    // Each group finishes a half of the parts: it leaves its sums of the other
    // half to the other group, a lane the ones of its own place.
    static_assert(kGroups == 2 && kMI % 2 == 0, "halves");
    const int at = wave * (kOwn * kNI * 64 * 16) + lane * 16;
#pragma unroll
    for (int i = 0; i < kOwn * kNI; ++i)
      *(f32x4*)(lds + at + i * 1024) = group ? acc[i / kNI][i % kNI]
                                             : acc[kOwn + i / kNI][i % kNI];
    arrived<0>();
    const char* theirs = lds_all + (1 - group) * kLds;
#pragma unroll
    for (int i = 0; i < kOwn * kNI; ++i) {
      f32x4& sum = acc[i / kNI][i % kNI];
      if (group) sum = acc[kOwn + i / kNI][i % kNI];
      sum += *(const f32x4*)(theirs + at + i * 1024);
    }
  }
  char* mine = lds + kSums + wave * (kParts * 16 * kCols * 4);
  const int own_m = m0 + xr + group * kOwn * 16;
  const int c = lane % kLanes, n = n0 + yr + c * kOut;
  constexpr int kTurns = kParts * 16 * kLanes / 64;        // of 64 lanes
  constexpr int kFetch = kTurns < 4 ? kTurns : 4;
  const int r_of_lane = lane / kLanes;
  const auto rows = [&](auto fetch, auto store) {
#pragma unroll
    for (int round = 0; round < kOwn / kParts; ++round) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const int r = i * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < kNI; ++j) {
          const int q = (j * 4 + (lane >> 4)) ^ (r & (kQuads - 1));
          *(f32x4*)(mine + (r * kQuads + q) * 16) =
              acc[round * kParts + i][j];
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int t0 = 0; t0 < kTurns; t0 += kFetch) {
        // What four rows need from memory is in flight before its first use.
        const int r0 = r_of_lane + t0 * (64 / kLanes);
        const int first_m = own_m + round * kParts * 16 + r0;
        decltype(fetch(0)) fetched[kFetch];
#pragma unroll
        for (int t = 0; t < kFetch; ++t) {
          const int m = first_m + t * (64 / kLanes);
          if (m < a.m && n < a.n) fetched[t] = fetch(m);
        }
#pragma unroll
        for (int t = 0; t < kFetch; ++t) {
          const int r = r0 + t * (64 / kLanes);
          const int m = first_m + t * (64 / kLanes);
          if (m >= a.m || n >= a.n) continue;
          float z[kOut];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int q = (c * 2 + h) ^ (r & (kQuads - 1));
            const f32x4 v = *(const f32x4*)(mine + (r * kQuads + q) * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[h * 4 + i] = v[i];
          }
          store(m, fetched[t], z);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (a.part != nullptr) {
    rows([](int) { return 0; }, [&](int m, int, float (&z)[kOut]) {
      store_f32<float, kOut>(
          a.part + ((long)split * a.m + m) * a.ld_part + n, z);
    });
    return;
  }
  float b[kOut];
  load_bias<T>(a.e, n, a.n, b);
  with_act(a.e.act, [&](auto act) {
    rows([&](int m) { return load_residual<T>(a.e, m, n, a.n); },
         [&](int m, Raw<T> r, float (&z)[kOut]) {
           finish<T, act>(a.e, m, n, a.n, b, r, z);
         });
  });
}

// Adds the splits' sums and finishes; one thread has 8 columns of a row.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(LinearProduct a) {
  const int across = a.ld_part / kOut;
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at >= (long)a.m * across) return;
  const long m = at / across;
  const int n = (int)(at % across) * kOut;
  const float* p = a.part + m * a.ld_part + n;
  float z[kOut], b[kOut];
  load_bias<T>(a.e, n, a.n, b);
  const Raw<T> r = load_residual<T>(a.e, m, n, a.n);
  load_f32<float, kOut>(p, z);
#pragma unroll 4
  for (int s = 1; s < a.splits; ++s) {
    float t[kOut];
    load_f32<float, kOut>(p + (long)s * a.m * a.ld_part, t);
#pragma unroll
    for (int i = 0; i < kOut; ++i) z[i] += t[i];
  }
  with_act(a.e.act,
           [&](auto act) { finish<T, act>(a.e, m, n, a.n, b, r, z); });
}

// --------------------------------------------------- dz, db and alignment

// dz = dy act'(z) (kAct) or dy with rows of ld_dz values, zeros past n;
// part: a row of column sums of the unrounded dz for each blockIdx.y. A
// thread has 8 columns, 32 threads a row; 8 rows at a time four deep, whose
// loads are all in flight.
template <typename T, bool kAct>
__global__ __launch_bounds__(256) void dz_kernel(
    const T* dy, const Kept<T>* slopes, T* dz, long second, float* part,
    int m, int n, long ld_dy, int ld_dz, int rows) {
  constexpr int kDeep = 4;
  __shared__ float lds[8][256 + 8];
  const int c = blockIdx.x * 256 + (threadIdx.x & 31) * 8;
  const int r0 = blockIdx.y * rows, r1 = r0 + rows < m ? r0 + rows : m;
  float sum[8] = {};
  for (int r = r0 + (threadIdx.x >> 5); r < r1; r += 8 * kDeep) {
    float g[kDeep][8];
    Kept<T> s[kDeep][8];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int row = r + 8 * d;
      const T* p = dy + row * ld_dy + c;
      const Kept<T>* q = slopes + (long)row * n + c;
      if (row >= r1) continue;
      load_some<T, 8>(p, n - c, g[d]);
      if (!kAct) continue;
      if (n - c >= 8) {
        __builtin_memcpy(s[d], q, sizeof(s[d]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[d][i] = i < n - c ? q[i] : Kept<T>{};
      }
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int row = r + 8 * d;
      if (row >= r1) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (kAct) g[d][i] *= kept<T>(s[d][i]);
        sum[i] += g[d][i];
      }
      if (dz) {
        T* out = dz + (long)row * ld_dz + c;
        store_some<T, 8>(out, ld_dz - c, g[d]);
        if (kAct && second) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float lost = g[d][i] - (float)(T)g[d][i];
            g[d][i] = __builtin_isfinite(lost) ? lost : 0.0f;
          }
          store_some<T, 8>(out + second, ld_dz - c, g[d]);
        }
      }
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    lds[threadIdx.x >> 5][(threadIdx.x & 31) * 8 + i] = sum[i];
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col < n) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += lds[i][threadIdx.x];
    part[(long)blockIdx.y * norm_part_half(n) + col] = t;
  }
}

// Rows of `width` values at any stride -> rows of `ld` values, a whole number
// of 16 bytes, zeros behind. A thread has 16 bytes of the result.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T* from, T* to,
                                                  int rows, int width,
                                                  long stride, int ld) {
  constexpr int kPer = 16 / sizeof(T);
  const int across = ld / kPer;
  const long total = (long)rows * across;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (long)gridDim.x * 256) {
    const long r = i / across;
    const int c = (int)(i % across) * kPer;
    const T* p = from + r * stride + c;
    T v[kPer];
    if (c + kPer <= width) {
      __builtin_memcpy(v, p, 16);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = c + j < width ? p[j] : (T)0.0f;
    }
    __builtin_memcpy(to + r * ld + c, v, 16);
  }
}

template <typename T, bool kXT, bool kYT, bool kTwo>
void run_tiles(const LinearProduct& a, hipStream_t s) {
  const unsigned grid = (unsigned)(((a.m + a.tile - 1) / a.tile) *
                                   ((a.n + a.tile - 1) / a.tile) * a.splits);
  if constexpr (sizeof(T) == 2) {
    if (a.tile == 256) {
      product_kernel<T, kXT, kYT, kTwo, 256, 256, 2, 4, 1, 2>
          <<<grid, 512, 0, s>>>(a);
      return;
    }
  }
  // A workgroup that has its CU to itself has two groups of waves, which halve
  // its steps, in place of one with more or more loads ahead: 64-wide bf16
  // 1024x1024x3999 22.3 -> 17.6 us and 100x1024x81 8.3 -> 7.2; 128-wide,
  // whose waves then read a quarter less LDS, 1024x1024x20000 in 4 splits
  // 53 -> 46, 1000x12544x1024 33 -> 31, few steps as before. Otherwise the
  // other workgroups' work covers its waits.
  if (a.tile == 128 && grid <= 256)
    product_kernel<T, kXT, kYT, kTwo, 128, 128, 2, 2, 2, 2>
        <<<grid, 512, 0, s>>>(a);
  else if (a.tile == 128)
    product_kernel<T, kXT, kYT, kTwo, 128, 128, 2, 4, 1, 2>
        <<<grid, 512, 0, s>>>(a);
  else if (grid <= 256)
    product_kernel<T, kXT, kYT, kTwo, 64, 64, 2, 2, 2, 4>
        <<<grid, 512, 0, s>>>(a);
  else
    product_kernel<T, kXT, kYT, kTwo, 64, 64, 2, 2, 1, 2>
        <<<grid, 256, 0, s>>>(a);
}

template <typename T>
hipError_t run_product(const LinearProduct& a, hipStream_t s) {
  constexpr bool parts = sizeof(T) == 2;     // fp32 has no second part
  if (!a.y_trans) run_tiles<T, false, false, false>(a, s);
  else if (a.x_trans && a.second) run_tiles<T, true, true, parts>(a, s);
  else if (a.x_trans) run_tiles<T, true, true, false>(a, s);
  else if (a.second) run_tiles<T, false, true, parts>(a, s);
  else run_tiles<T, false, true, false>(a, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.part == nullptr) return e;
  const long threads = (long)a.m * (a.ld_part / kOut);
  join_kernel<T><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t run_pad(const void* from, void* to, int rows, int width,
                   long stride, int ld, hipStream_t s) {
  const long blocks = ((long)rows * ld * sizeof(T) + 4095) / 4096;
  pad_kernel<T><<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, s>>>(
      (const T*)from, (T*)to, rows, width, stride, ld);
  return hipGetLastError();
}

}  // namespace

// The tile and the number of splits whose time is least by a model of what
// was measured on one MI355X (us): a step of a tile while all CUs work, what
// a tile takes besides its steps, and the splits' sums, written and read at
// 4.5 TB/s, with a second launch. Workgroups of a CU share it, so rounds are
// counted in CUs. For bf16 1000x12544x1024 it takes 4 splits of 128-wide
// tiles: 37 us, against 44 with 256-wide tiles in 12 splits and 43 with 3;
// for 32000 rows 256-wide ones unsplit: 617 us, against 845 with 128.
extern "C" bool linear_plan(LinearProduct* a, int type) {
  struct Shape { int tile; double step, alone, rest; };
  static const Shape kHalf[] = {{256, 1.55, 1.55, 6.0},
                                {128, 0.55, 0.48, 2.5},
                                {64, 0.25, 0.22, 1.0}};
  static const Shape kFull[] = {{128, 1.8, 1.8, 2.5}, {64, 0.5, 0.5, 1.0}};
  const Shape* shapes = type == kElemF32 ? kFull : kHalf;
  const int count = type == kElemF32 ? 2 : 3;
  const int per = type == kElemF32 ? 32 : 64;
  const int steps = (a->kx > per ? (a->kx + per - 1) / per : 1) *
                    (a->second ? 2 : 1);
  double best = 0.0;
  for (int i = 0; i < count; ++i) {
    const int t = shapes[i].tile;
    const long tiles = (long)((a->m + t - 1) / t) * ((a->n + t - 1) / t);
    // A launch has less than 2^32 threads, of 256 or 512 a tile (run_tiles).
    if (tiles >= 1L << (t == 64 ? 24 : 23)) continue;
    for (int s = 1; s <= 32 && (s == 1 || (s * 2 <= steps && tiles * s <= 2048));
         ++s) {
      const int each = (steps + s - 1) / s;
      const long rounds = (tiles * s + 255) / 256;
      const double us =
          rounds * (each * (rounds == 1 ? shapes[i].alone : shapes[i].step) +
                    shapes[i].rest) +
          (s > 1 ? 4.8 + (double)s * a->m * a->n * 8.0 / 4.5e6 : 0.0);
      if (best == 0.0 || us < best) {
        best = us;
        a->tile = t;
        a->steps_per_split = each;
        a->splits = (steps + each - 1) / each;
      }
    }
  }
  if (best == 0.0) return false;
  // Four rows of tiles by all columns at a time share more of both operands
  // in an L2 than one row does, once a row is longer than that.
  a->group = (a->n + a->tile - 1) / a->tile > 4 ? 4 : 1;
  a->ld_part = (a->n + kOut - 1) / kOut * kOut;
  return true;
}

extern "C" hipError_t linear_product_launch(const LinearProduct* a, int type,
                                            hipStream_t s) {
  switch (type) {
    case kElemF32: return run_product<float>(*a, s);
    case kElemBF16: return run_product<bf16_t>(*a, s);
    default: return run_product<fp16_t>(*a, s);
  }
}

extern "C" int linear_dz_strips(int m, int n) {
  const int across = (n + 255) / 256;
  int strips = 1024 / across;
  if (strips > (m + 31) / 32) strips = (m + 31) / 32;
  return strips < 1 ? 1 : strips;
}

template <typename T>
static hipError_t run_dz(const LinearDz& a, hipStream_t s) {
  const int rows = (a.m + a.strips - 1) / a.strips;
  const int cols = a.dz && a.ld_dz > a.n ? a.ld_dz : a.n;
  const dim3 grid((cols + 255) / 256, a.strips);
  const auto* kept = (const Kept<T>*)a.kept;
  if (kept != nullptr)
    dz_kernel<T, true><<<grid, 256, 0, s>>>((const T*)a.dy, kept, (T*)a.dz,
                                            a.second, a.part, a.m, a.n,
                                            a.ld_dy, a.ld_dz, rows);
  else
    dz_kernel<T, false><<<grid, 256, 0, s>>>((const T*)a.dy, kept, (T*)a.dz,
                                             0, a.part, a.m, a.n, a.ld_dy,
                                             a.ld_dz, rows);
  return hipGetLastError();
}

extern "C" hipError_t linear_dz_launch(const LinearDz* a, int type,
                                       hipStream_t s) {
  switch (type) {
    case kElemF32: return run_dz<float>(*a, s);
    case kElemBF16: return run_dz<bf16_t>(*a, s);
    default: return run_dz<fp16_t>(*a, s);
  }
}

extern "C" hipError_t linear_pad_launch(const void* from, void* to, int rows,
                                        int width, long stride, int ld,
                                        int type, hipStream_t s) {
  switch (type) {
    case kElemF32: return run_pad<float>(from, to, rows, width, stride, ld, s);
    case kElemBF16: return run_pad<bf16_t>(from, to, rows, width, stride, ld, s);
    default: return run_pad<fp16_t>(from, to, rows, width, stride, ld, s);
  }
}
