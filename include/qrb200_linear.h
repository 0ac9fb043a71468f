/*
 * qrb200_linear.h — C ABI of libqrb200.so, the linear-layer operators: the
 * matrix product with its epilogue, its backward pass (whose weight gradient
 * is the G of the statistics G G^T that qrb_gram_f32 forms), and activations
 * kept in 8 bits between the two.
 *
 * Conventions as in qrb200.h: device pointers, row-major matrices whose column
 * stride is 1 and whose row stride (ld*, in elements) is at least the row's
 * length, work enqueued on `stream` without synchronising, scratch passed in
 * by the caller, qrb_status codes, argument errors found on the host before
 * anything is enqueued. Outputs may not overlap inputs or one another, except
 * that qrbl_linear's y may be its residual (same address and row stride).
 *
 * Types: QRBL_F32, QRBL_F16 or QRBL_BF16 for every matrix and vector of one
 * call. Products accumulate in FP32 (FP16 and BF16 operands on the tensor
 * cores as they are, whose own sums, which do not round to nearest, are taken
 * out and added in FP32 after at most 8192 values: they add at most 2^-14 of
 * the terms' magnitudes to FP32's own roundings, at any length; FP32 operands as three BF16 parts
 * whose six largest products are formed, which keeps FP32's 24 bits of
 * operands above 2^-110 in magnitude; a product with an FP32 Inf may give NaN
 * instead of Inf). Every output is rounded once, to nearest even.
 *
 * Results are the same from call to call (no atomics), for given sizes,
 * alignments, device and set of arguments (what is asked for beside a product can
 * change how its reduction is cut, and so its last bits).
 */
#ifndef QRB200_LINEAR_H
#define QRB200_LINEAR_H

#include "qrb200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum { QRBL_F32 = 0, QRBL_F16 = 1, QRBL_BF16 = 2 };

/* Activations. GELU is z Phi(z); GELU_TANH its usual approximation
 * z / 2 (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))); SILU z / (1 + exp(-z)). */
enum { QRBL_ACT_NONE = 0, QRBL_ACT_RELU = 1, QRBL_ACT_GELU = 2, QRBL_ACT_GELU_TANH = 3,
       QRBL_ACT_SILU = 4 };

/*
 * The packed form of a matrix [rows, cols] of type t: codes int8 [rows, cols]
 * and exponents int8 [rows, ceil(cols / 32)], both contiguous. The values of
 * columns 32 j .. 32 j + 31 of a row share the step 2^e, e the smallest
 * integer with max |x| <= 127 * 2^e, clamped to [-126, 122] ([-24, 10] for
 * QRBL_F16) and at its lower end for a block of zeros; a code is x / 2^e
 * rounded to nearest even, at most 127 in magnitude (63 where e is at its
 * upper end), so that every value code * 2^e is exact in t. Inf and NaN do not
 * enter the maximum, get the code -128 and come back as NaN.
 */

/* Forward: z = x W^T + bias, y = act(z) + residual. */
typedef struct {
  int32_t dtype;
  int32_t activation;
  int64_t m, n, k;
  const void* x;         /* [m, k], row stride ldx */
  int64_t ldx;
  const void* w;         /* [n, k], row stride ldw */
  int64_t ldw;
  const void* bias;      /* [n] or NULL */
  const void* residual;  /* [m, n], row stride ldr, or NULL */
  int64_t ldr;
  void* y;               /* [m, n], row stride ldy */
  int64_t ldy;
  void* z;               /* [m, n], row stride ldz, or NULL: the pre-activation, kept */
  int64_t ldz;
  int8_t* z_codes;       /* [m, n], or NULL: the pre-activation, kept packed */
  int8_t* z_exponents;   /* [m, ceil(n / 32)]; given exactly when z_codes is */
} qrbl_linear_args;

/* Bytes of device workspace (16-byte aligned) qrbl_linear takes for these
 * arguments: operands that the tensor memory accelerator cannot read in
 * place (rows or base not 16-byte aligned; FP32 parts), the partial sums of
 * a product split along its reduction and the sums of a reduction longer
 * than 8192. A function of the arguments' sizes, strides, alignments and of
 * which pointers are given. 0 for invalid arguments. */
QRB_API size_t qrbl_linear_workspace_bytes(const qrbl_linear_args* args);
QRB_API int qrbl_linear(const qrbl_linear_args* args, void* workspace, size_t workspace_bytes,
                        void* stream);

/*
 * Backward: dz = dy * act'(z), dx = dz W, dw = dz^T x, dbias = column sums of
 * dz. (The residual's gradient is dy itself.) x and z each plain or packed; z
 * is not read with QRBL_ACT_NONE and otherwise required. With QRBL_ACT_RELU z
 * may not be packed: its derivative is the sign of z, which small values lose.
 * dz is rounded to the layer's type before the two products; dbias sums it
 * unrounded. Outputs that are NULL are not computed (x or w may then be NULL
 * where nothing needs them).
 */
typedef struct {
  int32_t dtype;
  int32_t activation;
  int64_t m, n, k;
  const void* dy;        /* [m, n], row stride lddy */
  int64_t lddy;
  const void* x;         /* [m, k], row stride ldx, or NULL */
  int64_t ldx;
  const int8_t* x_codes; /* packed x, or NULL */
  const int8_t* x_exponents;
  const void* w;         /* [n, k], row stride ldw */
  int64_t ldw;
  const void* z;         /* [m, n], row stride ldz, or NULL */
  int64_t ldz;
  const int8_t* z_codes; /* packed z, or NULL */
  const int8_t* z_exponents;
  void* dx;              /* [m, k], row stride lddx, or NULL */
  int64_t lddx;
  void* dw;              /* [n, k], row stride lddw, or NULL */
  int64_t lddw;
  void* dbias;           /* [n], or NULL */
} qrbl_linear_backward_args;

QRB_API size_t qrbl_linear_backward_workspace_bytes(const qrbl_linear_backward_args* args);
QRB_API int qrbl_linear_backward(const qrbl_linear_backward_args* args, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* A matrix [rows, cols] of type dtype, row stride ld, into its packed form and
 * back. */
QRB_API int qrbl_pack(int32_t dtype, const void* x, int64_t ld, int64_t rows, int64_t cols,
                      int8_t* codes, int8_t* exponents, void* stream);
QRB_API int qrbl_unpack(int32_t dtype, const int8_t* codes, const int8_t* exponents, int64_t rows,
                        int64_t cols, void* x, int64_t ld, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* QRB200_LINEAR_H */
