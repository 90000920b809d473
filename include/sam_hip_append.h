/*
 * sam_hip_append.h - new tokens into the paged memory with their position rotation, part of libsam_hip.so's C ABI. Conventions,
 * status codes and the switch are those of sam_hip.h, which includes this file.
 */
#ifndef SAM_HIP_APPEND_H
#define SAM_HIP_APPEND_H

#ifdef __cplusplus
extern "C" {
#endif

/*
 * What sam_hip_rope_axes of q and of k and sam_hip_kv_write (sam_hip_paged.h) do with new tokens, in one launch: q [tokens,
 * heads, d] turned goes to out, k [tokens, kv_heads, d] turned and v as it is into their pages, each token at the position
 * lens[b] - (starts[b+1] - t) of its sequence. Pair i (0 <= i < pairs) of a head turns by pos[t, axes[i]] * freqs[i] (a value of
 * axes outside 0 .. naxes - 1 takes position 0), or, with pos NULL, by the token's position in its sequence times freqs[i];
 * pairs are (x[2i], x[2i+1]) or, with halves, (x[i], x[i+pairs]); columns past 2 * pairs stay. No entry point of the
 * reference's corresponds to it: its memory attention projects, rotates and concatenates (sam3/video.rs:129-145, 356-406).
 *
 * A turned key is rounded once, to dtype or to its e4m3 or e2m1 codes (the turn is formed in f64; angles are exact to 2^-50 up
 * to 2^48 radians; beyond f32's largest number it is infinite); a turned query is formed in f32 and rounded to dtype. The cache,
 * its tables and what is checked on the device are those of sam_hip_kv_write. Rows of q that belong to no sequence stay as they
 * are in out, or become 0 with zero_rest; a token of a sequence that has no place in its pages still has its query turned.
 * q and out may both be NULL (heads is ignored then); with pairs == 0 pos, freqs and axes may be. Strides: (token, head) of q,
 * k, v and out in multiples of 16 bytes, (token, axis) of pos; NULL = contiguous; out's rows lie apart. out may be q with the
 * same strides; it must not overlap q otherwise, nor the other tensors. Limits: those of the paged memory, up to 65535 query
 * heads, tokens * (heads + kv_heads) <= 2^27 - 32.
 */
int sam_hip_kv_append(const void* q, const void* k, const void* v, const int* pos, const double* freqs, const int* axes,
                      void* out, void* k_pages, void* v_pages, unsigned char* k_scale, unsigned char* v_scale,
                      const int* table, const int* starts, const int* lens, int dtype, int cache_dtype, int tokens,
                      int batch, int heads, int pages, int kv_heads, int page_size, int d, int table_width, int pairs,
                      int naxes, const long* strides_q, const long* strides_k, const long* strides_v,
                      const long* strides_pos, const long* strides_out, int halves, int zero_rest, void* stream);

#ifdef __cplusplus
}
#endif
#endif
