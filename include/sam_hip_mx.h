/*
 * sam_hip_mx.h - microscaled 4-bit numbers, part of libsam_hip.so's C ABI. Conventions, status codes and the switch are
 * those of sam_hip.h, which includes this file.
 */
#ifndef SAM_HIP_MX_H
#define SAM_HIP_MX_H

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows of k values (k % 32 == 0) in blocks of 32, each value an e2m1 code (0 0.5 1 1.5 2 3 4 6 and their negatives) times
 * its block's scale 2^s, s the least integer within +-126 with max|x| <= 6 * 2^s (0 for a block of zeros), held as the
 * byte s + 127. codes [rows, k / 2]: two a byte, the even column's in the low half; scales [rows, k / 32]. A code is x / 2^s
 * rounded to the nearest e2m1, ties to even; a block with a value that is not finite has the scale byte 255 and is NaN
 * throughout. No entry point of the reference's corresponds to these: its linears (candle_nn::Linear, as in
 * sam1/encoder.rs:64) hold 16- or 32-bit weights.
 *
 * sam_hip_mx_pack writes the codes and scales of x [rows, k] in dtype; sam_hip_mx_unpack gives back the values that they
 * stand for, rounded to dtype once (a scale byte of 0 is 2^-127). At most 2^35 - 2048 values; x and
 * codes 16-byte aligned.
 */
int sam_hip_mx_pack(const void* x, unsigned char* codes, unsigned char* scales, int dtype, long rows, int k, void* stream);
int sam_hip_mx_unpack(const unsigned char* codes, const unsigned char* scales, void* x, int dtype, long rows, int k,
                      void* stream);

/*
 * out[i, j] = act(sum_l A[i, l] B[j, l] + bias[j]) over the values that a, a_scale [m, k] and b, b_scale [n, k] stand for:
 * a linear layer whose weights are B. Sums are f32, bias [n] (or NULL) and out [m, n] are of dtype, rounded once; act is the
 * identity or, with gelu, the exact GELU 0.5 x (1 + erf(x / sqrt 2)). out must not overlap the operands. m * n < 2^36,
 * m <= 2^30, n <= 2^25, k <= 2^22, fewer than 2^23 tiles of 128 x 128; a, b, bias and out 16-byte aligned. Rows whose
 * scales are no whole dwords (k % 128 != 0), and scales off a multiple of 4 bytes run slower.
 */
int sam_hip_mx_matmul(const unsigned char* a, const unsigned char* a_scale, const unsigned char* b,
                      const unsigned char* b_scale, const void* bias, void* out, int dtype, int m, int n, int k, int gelu,
                      void* stream);

/*
 * A linear layer with 4-bit weights: sam_hip_mx_pack of x [m, k] into the workspace, then sam_hip_mx_matmul of it and of w,
 * w_scale (as sam_hip_mx_pack makes them from [n, k]) to out [m, n]. Workspace: sam_hip_mx_linear_workspace_size() bytes of
 * device memory, 16-byte aligned (0 needs none, as a few rows are packed on their way to the product; -1 is an error; it depends
 * on the current device's CU count); calls that may overlap need their own, and so does each captured graph that may run beside
 * another.
 */
long sam_hip_mx_linear_workspace_size(int m, int n, int k);
int sam_hip_mx_linear(const void* x, const unsigned char* w, const unsigned char* w_scale, const void* bias, void* out,
                      int dtype, int m, int n, int k, int gelu, void* workspace, long workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
