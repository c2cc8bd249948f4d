// Arguments and launchers of the training operators, shared by their
// kernels (csrc/hip) and their bindings (csrc/train_ops.cpp).
#pragma once

#include <hip/hip_runtime.h>

// Host views of the tensors of one type; `ms` and `vs` are null with fp32
// states, `key` where 8-bit ones are rounded to nearest.
struct AdamWTensors {
  int count;
  void* const* p;
  const void* const* g;
  void* const* m;
  void* const* v;
  unsigned char* const* ms;
  unsigned char* const* vs;
  const unsigned* key;
  const long* n;
};

struct AdamWScalars {
  float beta1, one_minus_beta1, beta2, one_minus_beta2;
  float eps;
  float decay;         // 1 - lr * weight_decay
  float rate;          // lr / (1 - beta1^step)
  float inv_bc2;       // 1 / sqrt(1 - beta2^step)
  float max_norm;
  const float* norm;   // null: no clipping
};

// Sums of one row of partial sums: the width, a whole number of 16 bytes.
__host__ __device__ inline int norm_part_half(int width) {
  return (width + 3) / 4 * 4;
}

struct NormArgs {
  const void *dy, *x, *w, *b;     // w, b: null for 1 and 0
  void *y, *dx;
  float *mean, *rstd;
  float* part;         // `parts` rows of 2 * norm_part_half(width) sums
  long rows, x_stride, dy_stride;
  int width;
  int parts;           // the backward's grid
  float eps;
};

enum LinearAct : int { kActNone = 0, kActRelu, kActGelu, kActSilu };

struct LinearEpilogue {
  const void* bias;        // null: 0
  const void* residual;    // null: 0
  void* y;                 // rows of n values
  void* kept;              // act'(z) for the backward, rows of n values of
                           // fp32 or 16 bits as the tensors, or null
  long ld_residual;
  int act;
};

// D[m][n] = sum over k of X(m, k) Y(n, k). Rows of both operands begin at
// multiples of 16 bytes and their consecutive extent is a whole number of
// 16 bytes.
struct LinearProduct {
  const void *x, *y;
  long ldx, ldy;           // values between rows in memory
  long second;             // bytes from x to its second part, which is added
                           // to it (X = x + second part), or 0: it has one
  bool x_trans, y_trans;   // k is not the consecutive index
  int m, n;                // of D
  int ext_x, ext_y;        // of the operands in memory, m and n or padded
  int kx, ky;              // likewise of k
  // linear_plan()'s
  int tile, group, splits, steps_per_split, ld_part;
  float* part;             // splits * m * ld_part sums, or null (one split)
  LinearEpilogue e;
};

struct LinearDz {
  const void *dy, *kept;   // kept: of the epilogue, null: no activation
  void* dz;                // null: sums alone
  long second;             // values from dz to its second part, what the first
                           // one's rounding lost, or 0: none
  float* part;             // `strips` rows of norm_part_half(n) column sums,
                           // or null
  long ld_dy;
  int m, n, ld_dz, strips;
};

extern "C" {
bool linear_plan(LinearProduct*, int type);   // false: too large a launch
hipError_t linear_product_launch(const LinearProduct*, int type, hipStream_t);
int linear_dz_strips(int m, int n);
hipError_t linear_dz_launch(const LinearDz*, int type, hipStream_t);
// Rows of `width` values -> rows of `ld` values, a whole number of 16 bytes,
// zeros behind.
hipError_t linear_pad_launch(const void* from, void* to, int rows, int width,
                             long stride, int ld, int type, hipStream_t);

unsigned adamw_key(unsigned key, unsigned number);
hipError_t adamw_launch(const AdamWTensors*, const AdamWScalars*, int type,
                        hipStream_t);
// Values that one workgroup of square_sum_launch takes, of so many altogether.
int square_sum_chunk(long values);
// `partial` has a double for every chunk of every tensor.
hipError_t square_sum_launch(const void* const* g, const long* n, int count,
                             int chunk, int type, double* partial,
                             hipStream_t);
hipError_t norm_launch(const double* partial, int count, float* out,
                       hipStream_t);
hipError_t pack8_launch(const float* x, unsigned char* codes,
                        unsigned char* scales, long n, bool is_signed,
                        hipStream_t);
hipError_t unpack8_launch(const unsigned char* codes,
                          const unsigned char* scales, void* out, long n,
                          bool is_signed, int type, hipStream_t);

// Rows of partial sums that the norm's backward writes.
int layer_norm_parts(long rows, int width, int type);
hipError_t layer_norm_fwd_launch(const NormArgs*, int type, int wtype,
                                 hipStream_t);
hipError_t layer_norm_bwd_launch(const NormArgs*, int type, int wtype,
                                 hipStream_t);
// `count` rows of `cols` fp32 sums, cols % 4 == 0; the sums of columns
// 0 .. n - 1 go to out, of split .. split + n - 1 to out2; either may be null.
hipError_t sum_rows_launch(const float* part, int count, int cols, int split,
                           int n, void* out, void* out2, int type,
                           hipStream_t);
}
