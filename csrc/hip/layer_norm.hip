// Layer norm over the last dimension: forward, and the backward with the
// reduction of the weight's and bias's gradients.
//
//   mu = mean(x)   var = mean((x - mu)^2)   r = 1 / sqrt(var + eps)
//   xh = (x - mu) r           y = xh w + b
//   d = dy w       dx = r (d - mean(d) - xh mean(d xh))
//   dw = sum over rows of dy xh       db = sum over rows of dy
//
// Memory bound: x (and dy) are read once and stay in registers between the
// statistics and the result; the variance is taken from the differences to
// the mean, in fp32. A row belongs to a team of kTeam lanes (a part of a
// wave up to 64, a workgroup above), each holding kVecs packets of 16 bytes;
// a row may begin anywhere and its last packet may be a part of one.
// In the backward each lane also keeps its columns' sums of dy xh and dy
// over all rows it sees; they leave once per workgroup as one row of
// partial sums and a second launch adds the rows up in a fixed order, so
// the gradients do not change from run to run.
//
// Measured on one MI355X, where a copy reaches 4.9 to 5.4 TB/s: bf16
// 131072x256 forward 24 us (134 MB, 5.6 TB/s), backward 32 + 4 us for the
// partial sums' sum (201 MB); fp32 1000x12544 forward 20 us (100 MB, 5.0
// TB/s). Rows above 16384 values (2048 packets in 16 bits, 4096 in fp32) go to
// the wide kernels, which read x three times (mostly from the caches).
#include <hip/hip_runtime.h>

#include "train_ops.h"
#include "typed.h"

namespace {

// Sum over a team: within a wave by exchange, across waves through LDS.
// `lds` holds two floats a wave; the caller keeps calls apart with `slot`.
template <int kTeam>
__device__ inline float team_sum(float s, float* lds) {
  constexpr int in_wave = kTeam < 64 ? kTeam : 64;
#pragma unroll
  for (int d = in_wave / 2; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
  if constexpr (kTeam > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < kTeam / 64; ++w) s += lds[w];
  }
  return s;
}

template <int kTeam>
__device__ inline void team_sum2(float& a, float& b, float* lds) {
  constexpr int in_wave = kTeam < 64 ? kTeam : 64;
#pragma unroll
  for (int d = in_wave / 2; d >= 1; d >>= 1) {
    a += __shfl_xor(a, d, 64);
    b += __shfl_xor(b, d, 64);
  }
  if constexpr (kTeam > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      lds[threadIdx.x >> 6] = a;
      lds[16 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < kTeam / 64; ++w) {
      a += lds[w];
      b += lds[16 + w];
    }
  }
}

// Values of 16 bytes, what a lane moves at a time.
template <typename T>
constexpr int width_of() { return 16 / sizeof(T); }

template <int kTeam>
constexpr int threads_of() { return kTeam < 256 ? 256 : kTeam; }

// A packet of a row, of which `left` values are there if rows are ragged.
template <bool kRagged, typename T, int N>
__device__ inline void load_part(const T* p, int left, float (&out)[N]) {
  if constexpr (kRagged) load_some<T, N>(p, left, out);
  else load_f32<T, N>(p, out);
}

template <bool kRagged, typename T, int N>
__device__ inline void store_part(T* p, int left, const float (&in)[N]) {
  if constexpr (kRagged) store_some<T, N>(p, left, in);
  else store_f32<T, N>(p, in);
}

// T: x and y; W: weight and bias (null: 1 and 0).
template <typename T, typename W, int kTeam, int kVecs, bool kRagged>
__global__ __launch_bounds__(threads_of<kTeam>()) void norm_fwd_kernel(
    const T* x, const W* w, const W* b, T* y, float* mean, float* rstd,
    long rows, int width, long x_stride, float eps) {
  constexpr int kRows = threads_of<kTeam>() / kTeam;   // of one workgroup
  constexpr int kWidth = width_of<T>();
  __shared__ float lds[32];
  const long row = (long)blockIdx.x * kRows + threadIdx.x / kTeam;
  const int lane = threadIdx.x % kTeam;
  if (row >= rows) return;    // a whole team; above 64 lanes never part of one
  x += row * x_stride;
  y += row * (long)width;
  float v[kVecs][kWidth];
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int c = (k * kTeam + lane) * kWidth;
    if (c < width) {
      load_part<kRagged>(x + c, width - c, v[k]);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) s += v[k][i];
    }
  }
  const float inv = 1.0f / (float)width;
  const float mu = team_sum<kTeam>(s, lds) * inv;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int c = (k * kTeam + lane) * kWidth;
    if (c < width) {
#pragma unroll
      for (int i = 0; i < kWidth; ++i) {
        v[k][i] = !kRagged || c + i < width ? v[k][i] - mu : 0.0f;
        s += v[k][i] * v[k][i];
      }
    }
  }
  const float r = 1.0f / sqrtf(team_sum<kTeam>(s, lds) * inv + eps);
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int c = (k * kTeam + lane) * kWidth;
    if (c < width) {
      float wf[kWidth], bf[kWidth];
#pragma unroll
      for (int i = 0; i < kWidth; ++i) { wf[i] = 1.0f; bf[i] = 0.0f; }
      if (w != nullptr) load_part<kRagged>(w + c, width - c, wf);
      if (b != nullptr) load_part<kRagged>(b + c, width - c, bf);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) v[k][i] = v[k][i] * r * wf[i] + bf[i];
      store_part<kRagged>(y + c, width - c, v[k]);
    }
  }
  if (mean != nullptr && lane == 0) {
    mean[row] = mu;
    rstd[row] = r;
  }
}

// `part`: gridDim.x rows of two halves of sums (dy xh, then dy); null: no
// weight gradients wanted. `dx` may be null too.
template <typename T, typename W, int kTeam, int kVecs, bool kRagged>
__global__ __launch_bounds__(threads_of<kTeam>()) void norm_bwd_kernel(
    const T* dy, const T* x, const W* w, const float* mean, const float* rstd,
    T* dx, float* part, long rows, int width, long dy_stride, long x_stride) {
  constexpr int kThreads = threads_of<kTeam>();
  constexpr int kRows = kThreads / kTeam;
  constexpr int kWidth = width_of<T>();
  constexpr int kCols = kTeam * kVecs * kWidth;
  __shared__ float lds[32];
  __shared__ float sums[kRows > 1 ? 2 * kRows * kCols : 1];
  const int lane = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
  float wf[kVecs][kWidth], dw[kVecs][kWidth], db[kVecs][kWidth];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int c = (k * kTeam + lane) * kWidth;
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      wf[k][i] = 1.0f;
      dw[k][i] = db[k][i] = 0.0f;
    }
    if (w != nullptr && c < width)
      load_part<kRagged>(w + c, width - c, wf[k]);
  }
  const float inv = 1.0f / (float)width;
  for (long row = (long)blockIdx.x * kRows + team; row < rows;
       row += (long)gridDim.x * kRows) {
    const float mu = mean[row], r = rstd[row];
    const T* xr = x + row * x_stride;
    const T* dyr = dy + row * dy_stride;
    float d[kVecs][kWidth], xh[kVecs][kWidth];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kTeam + lane) * kWidth;
      if (c < width) {
        load_part<kRagged>(xr + c, width - c, xh[k]);
        load_part<kRagged>(dyr + c, width - c, d[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kTeam + lane) * kWidth;
      if (c < width) {
#pragma unroll
        for (int i = 0; i < kWidth; ++i) {
          xh[k][i] = (xh[k][i] - mu) * r;
          dw[k][i] += d[k][i] * xh[k][i];
          db[k][i] += d[k][i];
          d[k][i] *= wf[k][i];
          s1 += d[k][i];
          s2 += d[k][i] * xh[k][i];
        }
      }
    }
    if (dx == nullptr) continue;
    team_sum2<kTeam>(s1, s2, lds);
    s1 *= inv;
    s2 *= inv;
    T* dxr = dx + row * (long)width;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kTeam + lane) * kWidth;
      if (c < width) {
#pragma unroll
        for (int i = 0; i < kWidth; ++i)
          d[k][i] = r * (d[k][i] - s1 - xh[k][i] * s2);
        store_part<kRagged>(dxr + c, width - c, d[k]);
      }
    }
  }
  if (part == nullptr) return;
  const int pad = norm_part_half(width);
  part += (long)blockIdx.x * 2 * pad;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kTeam + lane) * kWidth;
      if (c < width) {
        store_part<kRagged>(part + c, width - c, dw[k]);
        store_part<kRagged>(part + pad + c, width - c, db[k]);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kTeam + lane) * kWidth;
#pragma unroll
      for (int i = 0; i < kWidth; ++i) {
        sums[team * kCols + c + i] = dw[k][i];
        sums[(kRows + team) * kCols + c + i] = db[k][i];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += kThreads) {
      float a = 0.0f, b = 0.0f;
#pragma unroll
      for (int t = 0; t < kRows; ++t) {
        a += sums[t * kCols + c];
        b += sums[(kRows + t) * kCols + c];
      }
      part[c] = a;
      part[pad + c] = b;
    }
  }
}

// ------------------------------------------- rows too wide for registers

constexpr int kWide = 1024;   // threads of one row

// f(column, values there) for the thread's packets of a row.
template <typename T, typename F>
__device__ inline void each_packet(int width, F f) {
  constexpr int kWidth = width_of<T>();
  for (int c = threadIdx.x * kWidth; c < width; c += kWide * kWidth)
    f(c, width - c);
}

template <typename T, typename W>
__global__ __launch_bounds__(kWide) void norm_fwd_wide_kernel(
    const T* x, const W* w, const W* b, T* y, float* mean, float* rstd,
    int width, long x_stride, float eps) {
  constexpr int kWidth = width_of<T>();
  __shared__ float lds[32];
  const long row = blockIdx.x;
  x += row * x_stride;
  y += row * (long)width;
  float s = 0.0f;
  each_packet<T>(width, [&](int c, int left) {
    float v[kWidth];
    load_some<T, kWidth>(x + c, left, v);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) s += v[i];
  });
  const float mu = team_sum<kWide>(s, lds) / (float)width;
  s = 0.0f;
  each_packet<T>(width, [&](int c, int left) {
    float v[kWidth];
    load_some<T, kWidth>(x + c, left, v);
#pragma unroll
    for (int i = 0; i < kWidth; ++i)
      s += i < left ? (v[i] - mu) * (v[i] - mu) : 0.0f;
  });
  const float r = 1.0f / sqrtf(team_sum<kWide>(s, lds) / (float)width + eps);
  each_packet<T>(width, [&](int c, int left) {
    float v[kWidth], wf[kWidth], bf[kWidth];
    load_some<T, kWidth>(x + c, left, v);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) { wf[i] = 1.0f; bf[i] = 0.0f; }
    if (w != nullptr) load_some<W, kWidth>(w + c, left, wf);
    if (b != nullptr) load_some<W, kWidth>(b + c, left, bf);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) v[i] = (v[i] - mu) * r * wf[i] + bf[i];
    store_some<T, kWidth>(y + c, left, v);
  });
  if (mean != nullptr && threadIdx.x == 0) {
    mean[row] = mu;
    rstd[row] = r;
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(kWide) void norm_dx_wide_kernel(
    const T* dy, const T* x, const W* w, const float* mean, const float* rstd,
    T* dx, int width, long dy_stride, long x_stride) {
  constexpr int kWidth = width_of<T>();
  __shared__ float lds[32];
  const long row = blockIdx.x;
  const float mu = mean[row], r = rstd[row];
  x += row * x_stride;
  dy += row * dy_stride;
  dx += row * (long)width;
  // d = dy w and xh of a packet; d is 0 past the row's end.
  const auto load = [&](int c, int left, float (&d)[kWidth],
                        float (&xh)[kWidth]) {
    load_some<T, kWidth>(dy + c, left, d);
    load_some<T, kWidth>(x + c, left, xh);
    float wf[kWidth];
#pragma unroll
    for (int i = 0; i < kWidth; ++i) wf[i] = 1.0f;
    if (w != nullptr) load_some<W, kWidth>(w + c, left, wf);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      d[i] *= wf[i];
      xh[i] = (xh[i] - mu) * r;
    }
  };
  float s1 = 0.0f, s2 = 0.0f;
  each_packet<T>(width, [&](int c, int left) {
    float d[kWidth], xh[kWidth];
    load(c, left, d, xh);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      s1 += d[i];
      s2 += d[i] * xh[i];
    }
  });
  team_sum2<kWide>(s1, s2, lds);
  s1 /= (float)width;
  s2 /= (float)width;
  each_packet<T>(width, [&](int c, int left) {
    float d[kWidth], xh[kWidth];
    load(c, left, d, xh);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) d[i] = r * (d[i] - s1 - xh[i] * s2);
    store_some<T, kWidth>(dx + c, left, d);
  });
}

// A packet of columns a thread, gridDim.y strips of rows.
template <typename T>
__global__ __launch_bounds__(256) void norm_dw_wide_kernel(
    const T* dy, const T* x, const float* mean, const float* rstd,
    float* part, long rows, int width, long dy_stride, long x_stride) {
  constexpr int kWidth = width_of<T>();
  const int c = (blockIdx.x * 256 + threadIdx.x) * kWidth;
  if (c >= width) return;
  float a[kWidth] = {}, b[kWidth] = {};
  for (long row = blockIdx.y; row < rows; row += gridDim.y) {
    const float mu = mean[row], r = rstd[row];
    float d[kWidth], v[kWidth];
    load_some<T, kWidth>(dy + row * dy_stride + c, width - c, d);
    load_some<T, kWidth>(x + row * x_stride + c, width - c, v);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      a[i] += d[i] * ((v[i] - mu) * r);
      b[i] += d[i];
    }
  }
  const int pad = norm_part_half(width);
  part += (long)blockIdx.y * 2 * pad + c;
  store_some<float, kWidth>(part, width - c, a);
  store_some<float, kWidth>(part + pad, width - c, b);
}

// --------------------------------------------------- partial sums' sum

// part: `count` rows of `cols` sums, cols % 4 == 0; columns 0 .. n - 1 go to
// out, split .. split + n - 1 to out2 (either may be null). A workgroup takes
// 64 columns, 16 lanes with 4 each; its 64 groups of lanes take every 64th
// row, four of them in flight. The order of the sums is fixed.
template <typename W>
__global__ __launch_bounds__(1024) void sum_rows_kernel(
    const float* part, int count, int cols, int split, int n, W* out,
    W* out2) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 15, strip = threadIdx.x >> 4;
  const int col = blockIdx.x * 64 + lane * 4;
  float s[4] = {};
  if (col < cols) {
    for (int i = strip; i < count; i += 256) {
      float t[4][4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + 64 * k < count)
          load_f32<float, 4>(part + (long)(i + 64 * k) * cols + col, t[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += t[k][j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s[j] += __shfl_xor(s[j], 16, 64);
    s[j] += __shfl_xor(s[j], 32, 64);
  }
  if ((threadIdx.x & 63) < 16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) lds[threadIdx.x >> 6][lane * 4 + j] = s[j];
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += lds[i][threadIdx.x];
  const int c = blockIdx.x * 64 + threadIdx.x;
  if (c < n && out != nullptr) out[c] = (W)sum;
  if (c >= split && c - split < n && out2 != nullptr) out2[c - split] = (W)sum;
}

}  // namespace

namespace {

// f(first row, rows) for as many rows at a time as a launch takes, which has
// less than 2^32 threads.
template <typename F>
void each_launch(long all, int threads, int per, F f) {
  const long most = (1L << 31) / threads * per;
  for (long at = 0; at < all; at += most)
    f(at, all - at < most ? all - at : most);
}

template <typename T, typename W, int kTeam, int kVecs, bool kRagged>
void run_team(const NormArgs& a, bool backward, hipStream_t s) {
  constexpr int threads = threads_of<kTeam>(), per = threads / kTeam;
  if (!backward) {
    each_launch(a.rows, threads, per, [&](long at, long rows) {
      const unsigned grid = (unsigned)((rows + per - 1) / per);
      norm_fwd_kernel<T, W, kTeam, kVecs, kRagged><<<grid, threads, 0, s>>>(
          (const T*)a.x + at * a.x_stride, (const W*)a.w, (const W*)a.b,
          (T*)a.y + at * a.width, a.mean ? a.mean + at : nullptr,
          a.rstd ? a.rstd + at : nullptr, rows, a.width, a.x_stride, a.eps);
    });
  } else {
    norm_bwd_kernel<T, W, kTeam, kVecs, kRagged><<<a.parts, threads, 0, s>>>(
        (const T*)a.dy, (const T*)a.x, (const W*)a.w, a.mean, a.rstd,
        (T*)a.dx, a.part, a.rows, a.width, a.dy_stride, a.x_stride);
  }
}

// Rows that one workgroup has in hand at a time.
int rows_at_once(int packets) {
  return packets <= 8 ? 32 : packets <= 16 ? 16 : packets <= 32 ? 8
         : packets <= 128 ? 4 : 1;
}

// A team is as small as its row allows, with few packets a lane: the
// exchange takes fewer steps and more rows are in flight.
template <typename T, typename W, bool kRagged>
bool run_width(const NormArgs& a, bool backward, hipStream_t s) {
  const int packets = (a.width + width_of<T>() - 1) / width_of<T>();
  if (packets <= 8) run_team<T, W, 8, 1, kRagged>(a, backward, s);
  else if (packets <= 16) run_team<T, W, 16, 1, kRagged>(a, backward, s);
  else if (packets <= 32) run_team<T, W, 32, 1, kRagged>(a, backward, s);
  else if (packets <= 64) run_team<T, W, 64, 1, kRagged>(a, backward, s);
  else if (packets <= 128) run_team<T, W, 64, 2, kRagged>(a, backward, s);
  else if (packets <= 256) run_team<T, W, 256, 1, kRagged>(a, backward, s);
  else if (packets <= 512) run_team<T, W, 256, 2, kRagged>(a, backward, s);
  else if (packets <= 1024) run_team<T, W, 256, 4, kRagged>(a, backward, s);
  else if (packets <= 2048) run_team<T, W, 512, 4, kRagged>(a, backward, s);
  else if (packets <= 4096) {
    // 1024 lanes have 128 registers each: the backward's four arrays of 32
    // values do not fit, so such rows go to the wide kernels.
    if constexpr (sizeof(T) == 4) {
      run_team<T, W, 1024, 4, kRagged>(a, backward, s);
    } else {
      return false;
    }
  } else {
    return false;
  }
  return true;
}

template <typename T, typename W>
void run_types(const NormArgs& a, bool backward, hipStream_t s) {
  if (a.width % width_of<T>() ? run_width<T, W, true>(a, backward, s)
                              : run_width<T, W, false>(a, backward, s))
    return;
  if (!backward) {
    each_launch(a.rows, kWide, 1, [&](long at, long rows) {
      norm_fwd_wide_kernel<T, W><<<(unsigned)rows, kWide, 0, s>>>(
          (const T*)a.x + at * a.x_stride, (const W*)a.w, (const W*)a.b,
          (T*)a.y + at * a.width, a.mean ? a.mean + at : nullptr,
          a.rstd ? a.rstd + at : nullptr, a.width, a.x_stride, a.eps);
    });
    return;
  }
  if (a.dx != nullptr)
    each_launch(a.rows, kWide, 1, [&](long at, long rows) {
      norm_dx_wide_kernel<T, W><<<(unsigned)rows, kWide, 0, s>>>(
          (const T*)a.dy + at * a.dy_stride, (const T*)a.x + at * a.x_stride,
          (const W*)a.w, a.mean + at, a.rstd + at, (T*)a.dx + at * a.width,
          a.width, a.dy_stride, a.x_stride);
    });
  if (a.part != nullptr)
    norm_dw_wide_kernel<T>
        <<<dim3((a.width + 256 * width_of<T>() - 1) / (256 * width_of<T>()),
                a.parts),
           256, 0, s>>>(
            (const T*)a.dy, (const T*)a.x, a.mean, a.rstd, a.part, a.rows,
            a.width, a.dy_stride, a.x_stride);
}

hipError_t run_norm(const NormArgs& a, int type, int wtype, bool backward,
                    hipStream_t s) {
  if (type == kElemF32) run_types<float, float>(a, backward, s);
  else if (type == kElemBF16 && wtype == kElemF32) run_types<bf16_t, float>(a, backward, s);
  else if (type == kElemBF16) run_types<bf16_t, bf16_t>(a, backward, s);
  else if (wtype == kElemF32) run_types<fp16_t, float>(a, backward, s);
  else run_types<fp16_t, fp16_t>(a, backward, s);
  return hipGetLastError();
}

}  // namespace

// Rows of partial sums that the backward writes, its workgroups: enough to
// fill the chip, few enough that their sums stay small beside x. Measured on
// one MI355X with 64 .. 2048 of them (us with the sums' sum): bf16
// 131072x256 71, 45, 38 and 44 at 256, 512, 1024 and 2048; 4000x4096 39, 28,
// 30 and 41; 1000x12544 37, 30, 38 and 54 at 128, 256, 512 and 1024; 500x30000
// 51, 55, 63 and 85 at 64, 128, 256 and 512.
extern "C" int layer_norm_parts(long rows, int width, int type) {
  const int per = type == kElemF32 ? 4 : 8;
  const int packets = (width + per - 1) / per;
  const int at_once = rows_at_once(packets);
  const long sets = (rows + at_once - 1) / at_once;
  const bool in_registers = packets <= (type == kElemF32 ? 4096 : 2048);
  const long most = !in_registers ? 64 : packets > 1024 ? 256
                    : packets > 512 ? 512 : 1024;
  return (int)(sets < most ? sets : most);
}

extern "C" hipError_t layer_norm_fwd_launch(const NormArgs* a, int type,
                                            int wtype, hipStream_t s) {
  return run_norm(*a, type, wtype, false, s);
}

extern "C" hipError_t layer_norm_bwd_launch(const NormArgs* a, int type,
                                            int wtype, hipStream_t s) {
  return run_norm(*a, type, wtype, true, s);
}

extern "C" hipError_t sum_rows_launch(const float* part, int count, int cols,
                                      int split, int n, void* out, void* out2,
                                      int type, hipStream_t s) {
  const unsigned grid = (unsigned)((cols + 63) / 64);
  switch (type) {
    case kElemF32: sum_rows_kernel<float><<<grid, 1024, 0, s>>>(part, count, cols, split, n, (float*)out, (float*)out2); break;
    case kElemBF16: sum_rows_kernel<bf16_t><<<grid, 1024, 0, s>>>(part, count, cols, split, n, (bf16_t*)out, (bf16_t*)out2); break;
    default: sum_rows_kernel<fp16_t><<<grid, 1024, 0, s>>>(part, count, cols, split, n, (fp16_t*)out, (fp16_t*)out2);
  }
  return hipGetLastError();
}
