// AdamW over many tensors in one launch, and the norm of many gradients.
//
//   c = min(1, max_norm / (|g| + 1e-6))          (1 without a norm)
//   m = b1 m + (1 - b1) (c g)
//   v = b2 v + (1 - b2) (c g)^2
//   p = p (1 - lr wd) - lr / bc1 * m / (sqrt(v) / sqrt(bc2) + eps)
//
// All of it in fp32; the scalars are formed in double on the host. With betas
// from 0.5 on the states are formed as m + (1 - b1) (c g - m), a difference
// and a fused product and sum: one rounding of the result, and that of a
// beta such as 0.999 to fp32, a fifth of a unit in the last place, leaves no
// trace. (With smaller betas the difference would cancel: there it is the
// products' sum, each rounded by itself.) The same in plain elementwise
// operations gives the states to the bit, and with them the same 8-bit codes.
// The update's root and quotient are the instructions' (1 unit in the last
// place each): 3 units of an update that is itself a small part of p, for a
// fifth of the 8-bit kernel's instructions.
//
// 8-bit states: 256 consecutive values of a tensor share a power of two
// 2^(E-127), the exponent of the largest magnitude among them, kept as one
// byte. A value is its ratio to that power with 3 bits of mantissa:
//   first moment   sign, 4 bits of exponent: 1.875 .. 2^-14, steps of 2^-17
//                  below
//   second moment  5 bits of exponent: 1.875 .. 2^-30, steps of 2^-33 below;
//                  a value above zero never gets the code of zero, because a
//                  zero in the denominator would blow the update up, while a
//                  value held too large only makes it smaller
// With a power of two as the scale the ratio is exact, and so is the held value
// in bf16. E = 255 (an infinity or NaN among the values) stands for NaN in the
// whole block.
//   Rounding to nearest (even) has the least error in one step; a ratio above
// 1.875 (up to 2) takes the top code, no further off than half a step. Over
// many steps it loses what moves a state by less than half a step of its code:
// codes lie 6 to 12% apart and a beta of 0.999 moves v down by 0.1% at most, so
// that v never falls and rises only on squares 34 to 63 times as large. With a
// seed the state is therefore rounded up or down at random, up with the
// probability of what lies above the lower code, so that its mean is the
// unrounded state's. A step adds at most |d| D to its variance (d the step's
// move, D the distance of two codes), which is a spread of about a quarter of
// v in the long run. What is rounded up past 1.875 takes 2 and with it the
// block's next exponent; else a block's largest value could not grow.
//   The random bits are an integer hash of the seed, the step, the tensor's
// number and the value's place: nothing is kept between calls, and the same
// call gives the same codes.
//
// Memory bound: 28 bytes a value with fp32 states and parameters, 16 with
// 8-bit states, some 60 and 120 vector instructions. One thread holds 4
// consecutive values (16-byte accesses; with 8-bit states a wave is exactly
// one block of 256, whose maximum is a wave reduction).
//
// Measured on one MI355X with the 63.8 million parameters of the 101-layer
// detector in fp32: the norm 55 us and the step 285 us (1.79 GB, 6.2 TB/s; a
// part of the gradients comes from the memory-side cache), 412 together
// before p, m and v went past the caches. With 8-bit states the step takes
// 195 us (1.02 GB, 5.3 TB/s), rounded to nearest; at random 3 to 5% more (196
// and 188 us where to nearest took 188 and 181 in turn with it).
#include <hip/hip_runtime.h>

#include "train_ops.h"
#include "typed.h"

namespace {

constexpr int kThreads = 256;
constexpr int kValues = 4;                       // consecutive, per thread
constexpr int kPass = kThreads * kValues;        // values of one pass
constexpr int kPasses = 4;                       // of one workgroup, or 1
constexpr int kNormPasses = 16, kNormFew = 4;    // the same of the norm's
constexpr int kBlock8 = 256;                     // values sharing a scale
static_assert(kPass % kBlock8 == 0 && kBlock8 == 64 * kValues,
              "a wave holds one block of an 8-bit state");

// Pointers travel as kernel arguments (below 4 KB), so a launch needs no
// copy to the device and can be captured.
constexpr int kTensors32 = 88, kTensors8 = 60, kTensorsNorm = 180;

template <int N>
struct Table32 {
  void* p[N];
  const void* g[N];
  void* m[N];
  void* v[N];
  long n[N];
  int first[N];     // first workgroup of the tensor
  int count, passes;
};

template <int N>
struct Table8 : Table32<N> {
  unsigned char* ms[N];
  unsigned char* vs[N];
  unsigned key[N];  // of the random bits
};

struct TableNorm {
  const void* g[kTensorsNorm];
  long n[kTensorsNorm];
  int first[kTensorsNorm];
  int count, passes;
};

// The last tensor whose first workgroup is not above `wg`: a lane compares
// one tensor's, all at a time, as the table is far away.
template <typename Table>
__device__ inline int find_tensor(const Table& t, int wg) {
  constexpr int most = sizeof(t.first) / sizeof(t.first[0]);
  int k = -1;
#pragma unroll
  for (int i = 0; i < most; i += 64) {
    const int at = i + (threadIdx.x & 63);
    const int first = t.first[at < most ? at : most - 1];
    k += __popcll(__ballot(at < t.count && first <= wg));
  }
  return __builtin_amdgcn_readfirstlane(k);
}

struct Hyper {
  float beta1, one_minus_beta1, beta2, one_minus_beta2;
  float eps, decay, rate, inv_bc2, max_norm;
  const float* norm;       // null: no clipping
};

__device__ inline float clip_factor(const Hyper& h) {
  if (h.norm == nullptr) return 1.0f;
  const float c = h.max_norm / (*h.norm + 1e-6f);
  return c > 1.0f ? 1.0f : c;                    // NaN stays NaN
}

// The root, 0 and subnormal arguments (which the instruction takes for 0)
// too.
__device__ inline float root(float v) {
  const bool tiny = v < 0x1p-96f;
  const float s = __builtin_amdgcn_sqrtf(tiny ? v * 0x1p64f : v);
  return tiny ? s * 0x1p-32f : s;
}

// The state after `in`; where it may be one (k32), an overflown state stays.
template <bool kLerp, bool k32>
__device__ inline float moved(float state, float in, float beta,
                              float one_minus) {
#pragma clang fp contract(off)
  if constexpr (!kLerp) return state * beta + in * one_minus;
  const float d = in - state;
  const float x = __builtin_fmaf(d, one_minus, state);
  return k32 && __builtin_isinf(state) ? state + in : x;
}

template <bool kLerp, bool k32>
__device__ inline void update(const Hyper& h, float c, float g, float& p,
                              float& m, float& v) {
#pragma clang fp contract(off)
  g = g * c;
  m = moved<kLerp, k32>(m, g, h.beta1, h.one_minus_beta1);
  v = moved<kLerp, k32>(v, g * g, h.beta2, h.one_minus_beta2);
  const float step =
      m * __builtin_amdgcn_rcpf(root(v) * h.inv_bc2 + h.eps);
  p = p * h.decay - step * h.rate;
}

// Workgroups go through the tensors from the end: the norm, if there is one,
// has just read the gradients from the beginning, and the last of them are
// still in the memory-side cache.
template <typename Table>
__device__ inline int turned(const Table&) {
  return gridDim.x - 1 - blockIdx.x;
}

template <typename T, bool kLerp>
__global__ __launch_bounds__(kThreads) void adamw32_kernel(
    Table32<kTensors32> t, Hyper h) {
  const int wg = turned(t), k = find_tensor(t, wg);
  const long at = (long)(wg - t.first[k]) * t.passes * kPass +
                  threadIdx.x * kValues;
  const long n = t.n[k];
  T* p = static_cast<T*>(t.p[k]);
  const T* g = static_cast<const T*>(t.g[k]);
  float* m = static_cast<float*>(t.m[k]);
  float* v = static_cast<float*>(t.v[k]);
  const float c = clip_factor(h);
  for (int pass = 0; pass < t.passes; ++pass) {
    const long i = at + (long)pass * kPass, left = n - i;
    if (left <= 0) return;
    float pf[kValues], gf[kValues], mf[kValues], vf[kValues];
    stream_in(p + i, left, pf);
    stream_in(g + i, left, gf);
    stream_in(m + i, left, mf);
    stream_in(v + i, left, vf);
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      update<kLerp, true>(h, c, gf[j], pf[j], mf[j], vf[j]);
    stream_out(p + i, left, pf);
    stream_out(m + i, left, mf);
    stream_out(v + i, left, vf);
  }
}

// ---------------------------------------------------------- 8-bit states

__device__ inline float pow2_biased(int e) {     // 2^(e - 127), 1 <= e <= 254
  return __int_as_float(e << 23);
}

// kLow: the exponent of the smallest normal code is -kLow.
template <bool kSigned> struct Code8;
template <> struct Code8<true> { static constexpr int low = 14, top = 127; };
template <> struct Code8<false> { static constexpr int low = 30, top = 255; };

constexpr int kMinExp = 40;  // keeps 2^(E-127) and every step a normal fp32

// 2^(E - 127), NaN for E = 255.
__device__ inline float scale8(int e) {
  return e == 255 ? __int_as_float(0x7fc00000) : pow2_biased(e);
}

// A hash of 32 bits: products with odd numbers and shifts, each of them a
// permutation, so that every input bit changes every output bit in half of
// all cases (to the 1% that 16384 inputs can tell). ops/adamw.py has it too.
__host__ __device__ inline unsigned mix(unsigned x) {
  x = (x ^ x >> 16) * 0xac9b39d5u;
  x = (x ^ x >> 15) * 0x8fe44835u;
  return x ^ x >> 16;
}

// A code in the place of an fp32 number's exponent and first 3 bits is its
// value times a power of two, the codes below the smallest normal one being
// subnormal there too.
template <bool kSigned>
__device__ inline float decode8(unsigned code, float scale) {
  constexpr int low = Code8<kSigned>::low;
  const float r =
      __uint_as_float((kSigned ? code & 127u : code) << 20) *
      pow2_biased(127 + 126 - low) * scale;
  return kSigned && code > 127 ? -r : r;
}

// A number whose first 3 bits of mantissa are all there is, from x's magnitude
// and 20 random bits: up with the probability of what is cut off. Infinities
// and NaN stay in the largest exponent, and nothing else gets there.
__device__ inline float cut(float x, unsigned bits) {
  const unsigned b = __float_as_uint(x), mag = b & 0x7fffffffu;
  const unsigned up = mag + bits;
  return __uint_as_float(((up < 0x7f800000u ? up : mag) & 0x7ff00000u) |
                         (b & 0x80000000u));
}

// `inv` = 2^(127 - E). kRandom: x is cut()'s, and `hash` gives the bits where
// a small code has fewer than 3 of mantissa; `above`: the state is above zero.
template <bool kSigned, bool kRandom>
__device__ inline unsigned encode8(float x, float inv, bool above,
                                   unsigned hash) {
  constexpr int low = Code8<kSigned>::low;
  const float r = fabsf(x) * inv;
  const int b = __float_as_int(r);
  int code = ((b + 0x7ffff + ((b >> 20) & 1)) >> 20) - ((126 - low) << 3);
  code = code > Code8<kSigned>::top ? Code8<kSigned>::top : code;
  const bool small = r < pow2_biased(127 - low);
  if (__any(small)) {                  // rare but for zeros
    const float q = r * pow2_biased(127 + low + 3);
    int c;
    if constexpr (kRandom) {
      const float whole = floorf(q);
      const unsigned u = mix(hash + (kSigned ? 1 : 2)) >> 8;
      c = (int)whole + ((float)u * 0x1p-24f < q - whole);
    } else {
      c = (int)rintf(q);
    }
    if (!kSigned && above && c == 0) c = 1;   // also where r is 0
    code = small ? c : code;
  }
  if (kSigned) code |= (int)(__float_as_uint(x) >> 24) & 128;
  return (unsigned)code;
}

// The block's biased exponent from the largest magnitude's bits: as an
// unsigned maximum it lets infinities and NaN win.
__device__ inline int block_exponent(const float (&x)[kValues]) {
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
    const unsigned b = __float_as_uint(x[j]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const unsigned o = __shfl_xor(top, d, 64);
    top = o > top ? o : top;
  }
  const int e = (int)(top >> 23);
  return e < kMinExp ? kMinExp : e;
}

// kRandom: `hash` has 20 bits for each moment, the first's the lower ones. (The
// second's last 8 are the first's first 8, far too small a part to tell.)
template <bool kSigned, bool kRandom>
__device__ inline void store_block8(unsigned char* codes, unsigned char* scale,
                                    long left, const float (&x)[kValues],
                                    const unsigned (&hash)[kValues]) {
  float y[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j)
    y[j] = !kRandom ? x[j]
           : cut(x[j], kSigned ? hash[j] & 0xfffffu : hash[j] >> 12);
  const int e = block_exponent(y);
  unsigned c[kValues] = {};
  if (e < 255) {                       // of the whole wave
    const float inv = __int_as_float(e < 254 ? (254 - e) << 23 : 0x400000);
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      c[j] = encode8<kSigned, kRandom>(y[j], inv, x[j] > 0.0f, hash[j]);
  }
  if (left >= kValues) {
    const unsigned w = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
    __builtin_memcpy(codes, &w, 4);
  } else {
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      if (j < left) codes[j] = (unsigned char)c[j];
  }
  if ((threadIdx.x & 63) == 0 && left > 0) *scale = (unsigned char)e;
}

// Four codes as they lie in memory, zeros past the end.
__device__ inline unsigned load_codes(const unsigned char* codes, long left) {
  unsigned w = 0;
  if (left >= kValues) {
    __builtin_memcpy(&w, codes, 4);
    return w;
  }
#pragma unroll
  for (int j = 0; j < kValues; ++j)
    if (j < left) w |= (unsigned)codes[j] << (8 * j);
  return w;
}

template <bool kSigned>
__device__ inline void decode_block8(unsigned w, int e, float (&x)[kValues]) {
  const float scale = scale8(e);
#pragma unroll
  for (int j = 0; j < kValues; ++j)
    x[j] = decode8<kSigned>((w >> (8 * j)) & 255u, scale);
}

// 0 for a number in the middle between two codes.
__device__ inline unsigned middle(float x) {
  return (__float_as_uint(x) << 12) + 0x80000000u;
}

// x = moved(state, in) in such a middle goes by its last bit to where it was
// before its rounding, so that its code is that of the unrounded state. (The
// difference to the old state loses a last bit at most, far below what was
// rounded off.)
__device__ inline void leave_middle(float& x, float state, float in,
                                    float one_minus) {
#pragma clang fp contract(off)
  if (middle(x) != 0) return;
  const float lost = __builtin_fmaf(in - state, one_minus, state - x);
  const int up = lost == 0.0f ? 0 : (lost > 0.0f) == (x > 0.0f) ? 1 : -1;
  x = __int_as_float(__float_as_int(x) + up);
}

// One pass at a time: 60 registers, so that eight waves of a SIMD cover each
// other's loads. Two at a time took 92 registers, and 143 us in place of 125
// for 48 million values.
template <typename T, bool kLerp, bool kRandom>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(
    Table8<kTensors8> t, Hyper h) {
  const int wg = turned(t), k = find_tensor(t, wg);
  const long at = (long)(wg - t.first[k]) * t.passes * kPass +
                  threadIdx.x * kValues;
  const long n = t.n[k];
  T* p = static_cast<T*>(t.p[k]);
  const T* g = static_cast<const T*>(t.g[k]);
  unsigned char* m = static_cast<unsigned char*>(t.m[k]);
  unsigned char* v = static_cast<unsigned char*>(t.v[k]);
  unsigned char* ms = t.ms[k];
  unsigned char* vs = t.vs[k];
  const float c = clip_factor(h);
  for (int pass = 0; pass < t.passes; ++pass) {
    const long i = at + (long)pass * kPass, left = n - i;
    const long b = i / kBlock8;
    // A wave is past its end as a whole: it has one block.
    if (b * kBlock8 >= n) return;
    float pf[kValues], gf[kValues], mf[kValues], vf[kValues];
    stream_in(p + i, left, pf);
    stream_in(g + i, left, gf);
    const unsigned mc = load_codes(m + i, left), vc = load_codes(v + i, left);
    const unsigned me = ms[b], ve = vs[b];
    decode_block8<true>(mc, me, mf);
    decode_block8<false>(vc, ve, vf);
    unsigned between = 1;
#pragma unroll
    for (int j = 0; j < kValues; ++j) {
      update<kLerp, false>(h, c, gf[j], pf[j], mf[j], vf[j]);
      between = min(between, min(middle(mf[j]), middle(vf[j])));
    }
    if (!kRandom && kLerp && between == 0) {   // one wave in a few thousand
      float m0[kValues], v0[kValues];
      decode_block8<true>(mc, me, m0);
      decode_block8<false>(vc, ve, v0);
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        const float in = gf[j] * c;
        leave_middle(mf[j], m0[j], in, h.one_minus_beta1);
        leave_middle(vf[j], v0[j], in * in, h.one_minus_beta2);
      }
    }
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      if (j >= left) mf[j] = vf[j] = 0.0f;   // no part in the maximum
    unsigned hash[kValues] = {};
    if constexpr (kRandom) {
      const unsigned key = t.key[k] ^ (unsigned)(i >> 32) * 0x8fe44835u;
#pragma unroll
      for (int j = 0; j < kValues; ++j) hash[j] = mix((unsigned)i + j ^ key);
    }
    stream_out(p + i, left, pf);
    store_block8<true, kRandom>(m + i, ms + b, left, mf, hash);
    store_block8<false, kRandom>(v + i, vs + b, left, vf, hash);
  }
}

// ------------------------------------------------- packing and unpacking

template <bool kSigned>
__global__ __launch_bounds__(kThreads) void pack8_kernel(
    const float* x, unsigned char* codes, unsigned char* scales, long n) {
  const long i = ((long)blockIdx.x * kThreads + threadIdx.x) * kValues;
  const long b = i / kBlock8, left = n - i;
  if (b * kBlock8 >= n) return;
  float f[kValues];
  load_some(x + i, left, f);
  store_block8<kSigned, false>(codes + i, scales + b, left, f, {});
}

// 16 bytes of the result a thread, four times: a wave's accesses lie together,
// and past the caches no line is written in parts. (The result is larger than
// what the caches should give up for it.)
constexpr int kUnpackTimes = 4;
template <typename T>
constexpr int unpack_of() { return kUnpackTimes * kThreads * (16 / (int)sizeof(T)); }

template <bool kSigned, typename T>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(
    const unsigned char* codes, const unsigned char* scales, T* out, long n) {
  constexpr int kStore = 16 / sizeof(T);
  const long first = (long)blockIdx.x * unpack_of<T>() + threadIdx.x * kStore;
#pragma unroll
  for (int d = 0; d < kUnpackTimes; ++d) {
    const long i = first + d * kThreads * kStore;
    if (i >= n) return;
    const float e = scale8(scales[i / kBlock8]);
    float f[kStore];
    load_some<unsigned char, kStore>(codes + i, n - i, f);
#pragma unroll
    for (int j = 0; j < kStore; ++j) f[j] = decode8<kSigned>((unsigned)f[j], e);
    stream_out<T, kStore>(out + i, n - i, f);
  }
}

// ------------------------------------------------------------------ norm

// Squares are summed in double: memory bound all the same, and the result
// does not depend on the order to any bit of the fp32 norm that matters.
// Four loads of a thread are in flight.
template <typename T>
__global__ __launch_bounds__(kThreads) void square_sum_kernel(
    TableNorm t, double* partial) {
  constexpr int kDeep = 4;
  static_assert(kNormPasses % kDeep == 0 && kNormFew % kDeep == 0,
                "whole rounds");
  const int k = find_tensor(t, blockIdx.x);
  const long at = (long)(blockIdx.x - t.first[k]) * t.passes * kPass +
                  threadIdx.x * kValues;
  const long n = t.n[k];
  const T* g = static_cast<const T*>(t.g[k]);
  double s = 0.0;
  for (int pass = 0; pass < t.passes; pass += kDeep) {
    const long i = at + (long)pass * kPass;
    if (i >= n) break;
    float f[kDeep][kValues];
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
      load_some(g + i + d * kPass, n - i - d * kPass, f[d]);
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
#pragma unroll
      for (int j = 0; j < kValues; ++j)
        s += (double)f[d][j] * (double)f[d][j];
  }
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
  __shared__ double waves[kThreads / 64];
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) s += waves[w];
    partial[blockIdx.x] = s;
  }
}

__global__ __launch_bounds__(1024) void norm_kernel(const double* partial,
                                                    int count, float* out) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) s += partial[i];
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
  __shared__ double waves[16];
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += waves[w];
    *out = (float)sqrt(s);
  }
}

int chunks(long n, long each) { return (int)((n + each - 1) / each); }

}  // namespace

// Tensors from .. to - 1; returns the number of workgroups.
template <typename Table>
static int fill(Table& t, const AdamWTensors& a, int from, int to,
                int passes) {
  int wg = 0;
  t.count = to - from;
  t.passes = passes;
  for (int i = from; i < to; ++i) {
    const int k = i - from;
    t.p[k] = a.p[i];
    t.g[k] = a.g[i];
    t.m[k] = a.m[i];
    t.v[k] = a.v[i];
    t.n[k] = a.n[i];
    t.first[k] = wg;
    wg += chunks(a.n[i], (long)passes * kPass);
  }
  return wg;
}

template <typename T, bool kLerp>
static hipError_t run_adamw(const AdamWTensors& a, const Hyper& h,
                            hipStream_t stream) {
  const int most = a.ms == nullptr ? kTensors32 : kTensors8;
  for (int to = a.count; to > 0;) {
    const int from = to > most ? to - most : 0;
    // Four passes a workgroup amortise its search for the tensor; few values
    // are spread over more workgroups instead.
    long values = 0;
    for (int i = from; i < to; ++i) values += a.n[i];
    const int passes = values >= 1024L * kPasses * kPass ? kPasses : 1;
    if (a.ms == nullptr) {
      Table32<kTensors32> t;
      const int wg = fill(t, a, from, to, passes);
      adamw32_kernel<T, kLerp><<<wg, kThreads, 0, stream>>>(t, h);
    } else {
      Table8<kTensors8> t;
      const int wg = fill(t, a, from, to, passes);
      for (int i = from; i < to; ++i) {
        t.ms[i - from] = a.ms[i];
        t.vs[i - from] = a.vs[i];
        t.key[i - from] = a.key ? a.key[i] : 0;
      }
      if (a.key)
        adamw8_kernel<T, kLerp, true><<<wg, kThreads, 0, stream>>>(t, h);
      else
        adamw8_kernel<T, kLerp, false><<<wg, kThreads, 0, stream>>>(t, h);
    }
    to = from;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <bool kLerp>
static hipError_t run_adamw(const AdamWTensors& a, const Hyper& h, int type,
                            hipStream_t stream) {
  switch (type) {
    case kElemF32: return run_adamw<float, kLerp>(a, h, stream);
    case kElemBF16: return run_adamw<bf16_t, kLerp>(a, h, stream);
    default: return run_adamw<fp16_t, kLerp>(a, h, stream);
  }
}

// A number's 32 bits after 32 others; the numbers in turn give a tensor's key.
extern "C" unsigned adamw_key(unsigned key, unsigned number) {
  return mix(key + number + 0xac9b39d5u);
}

extern "C" hipError_t adamw_launch(const AdamWTensors* a,
                                   const AdamWScalars* s, int type,
                                   hipStream_t stream) {
  const Hyper h{s->beta1, s->one_minus_beta1, s->beta2, s->one_minus_beta2,
                s->eps, s->decay, s->rate, s->inv_bc2, s->max_norm, s->norm};
  return s->beta1 >= 0.5f && s->beta2 >= 0.5f
             ? run_adamw<true>(*a, h, type, stream)
             : run_adamw<false>(*a, h, type, stream);
}

// Values of one partial sum. Few values altogether are spread over more
// workgroups: 0.4 million take 3.6 us in place of 5.5.
extern "C" int square_sum_chunk(long values) {
  return (values >= 1024L * kNormPasses * kPass ? kNormPasses : kNormFew) *
         kPass;
}

extern "C" hipError_t square_sum_launch(const void* const* g, const long* n,
                                        int count, int chunk, int type,
                                        double* partial, hipStream_t stream) {
  for (int from = 0; from < count;) {
    TableNorm t;
    t.passes = chunk / kPass;
    int wg = 0;
    for (t.count = 0; from < count && t.count < kTensorsNorm; ++from) {
      const int k = t.count++;
      t.g[k] = g[from];
      t.n[k] = n[from];
      t.first[k] = wg;
      wg += chunks(n[from], chunk);
    }
    switch (type) {
      case kElemF32: square_sum_kernel<float><<<wg, kThreads, 0, stream>>>(t, partial); break;
      case kElemBF16: square_sum_kernel<bf16_t><<<wg, kThreads, 0, stream>>>(t, partial); break;
      default: square_sum_kernel<fp16_t><<<wg, kThreads, 0, stream>>>(t, partial);
    }
    partial += wg;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

extern "C" hipError_t norm_launch(const double* partial, int count, float* out,
                                  hipStream_t stream) {
  norm_kernel<<<1, 1024, 0, stream>>>(partial, count, out);
  return hipGetLastError();
}

extern "C" hipError_t pack8_launch(const float* x, unsigned char* codes,
                                   unsigned char* scales, long n,
                                   bool is_signed, hipStream_t stream) {
  constexpr long most = 1L << 33;     // a launch has less than 2^32 threads
  for (; n > 0; n -= most, x += most, codes += most,
                scales += most / kBlock8) {
    const long some = n < most ? n : most;
    const unsigned wg = (unsigned)((some + kPass - 1) / kPass);
    if (is_signed)
      pack8_kernel<true><<<wg, kThreads, 0, stream>>>(x, codes, scales, some);
    else
      pack8_kernel<false><<<wg, kThreads, 0, stream>>>(x, codes, scales, some);
  }
  return hipGetLastError();
}

template <bool kSigned>
static void unpack8(const unsigned char* codes, const unsigned char* scales,
                    void* out, long n, int type, hipStream_t stream) {
  const unsigned wg = (unsigned)chunks(
      n, type == kElemF32 ? unpack_of<float>() : unpack_of<bf16_t>());
  switch (type) {
    case kElemF32: unpack8_kernel<kSigned, float><<<wg, kThreads, 0, stream>>>(codes, scales, (float*)out, n); break;
    case kElemBF16: unpack8_kernel<kSigned, bf16_t><<<wg, kThreads, 0, stream>>>(codes, scales, (bf16_t*)out, n); break;
    default: unpack8_kernel<kSigned, fp16_t><<<wg, kThreads, 0, stream>>>(codes, scales, (fp16_t*)out, n);
  }
}

extern "C" hipError_t unpack8_launch(const unsigned char* codes,
                                     const unsigned char* scales, void* out,
                                     long n, bool is_signed, int type,
                                     hipStream_t stream) {
  if (is_signed) unpack8<true>(codes, scales, out, n, type, stream);
  else unpack8<false>(codes, scales, out, n, type, stream);
  return hipGetLastError();
}
