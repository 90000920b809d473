/*
 * sam_hip_paged.h - the paged memory's part of libsam_hip.so's C ABI. Conventions, status codes and the switch are those
 * of sam_hip.h, which includes this file.
 */
#ifndef SAM_HIP_PAGED_H
#define SAM_HIP_PAGED_H

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The paged memory: rotary positions over several axes, a cache of keys and values in pages, and the attention of new
 * tokens over it. The reference gathers its video memory into one tensor and rotates every key again on each frame
 * (sam3/video.rs:133-145, 356-406); here a frame's keys are rotated and stored once, in 16, 8 or 4 bits, and sequences
 * (tracked objects, say) of different lengths are read through their page tables. No entry point of the reference's
 * corresponds to these five.
 *
 * Rotary positions: pair i (0 <= i < pairs) of each head of x [b, l, h, d] turns by the angle pos[.., axes[i]] * freqs[i],
 *   y0 = x0 cos - x1 sin, y1 = x1 cos + x0 sin,
 * for (x0, x1) = (x[2i], x[2i+1]) or, with halves, (x[i], x[i + pairs]); columns past 2 * pairs are copied. inverse
 * turns by the negative angle (the gradient's way back). pos [b, l, naxes] int32 with strides (batch, token, axis), 0 to
 * share positions; freqs [pairs] f64, radians per unit of position; axes [pairs] int32 in [0, naxes) (another value
 * takes position 0); with pairs == 0 all three may be NULL. The angle is formed in f64, sine, cosine and the turn in
 * f32. Strides of x and out: (batch, token, head) elements, NULL = contiguous; the head dimension is contiguous. out's
 * rows lie apart; out may be x with the same strides and must not overlap x otherwise. Pointers are aligned to their
 * elements; 16-byte aligned rows with pairs % 4 == 0 (halves: pairs % 8 == 0) run on the vector kernel. Fewer than 2^31
 * tokens and 2^31 - 256 elements of one, up to 65535 heads and 2^38 elements.
 */
int sam_hip_rope_axes(const void* x, const int* pos, const double* freqs, const int* axes, void* out, int dtype, int b,
                      int l, int h, int d, int pairs, int naxes, const long* strides_x, const long* strides_pos,
                      const long* strides_out, int halves, int inverse, void* stream);

/*
 * The cache. k_pages and v_pages are pools [pages, kv_heads, page_size, d], contiguous and 16-byte aligned, of the call's
 * dtype, or of e4m3 (cache_dtype SAM_HIP_E4M3) with scales k_scale, v_scale [pages, kv_heads, page_size] of one byte. Key
 * j of sequence b lies in page table[b][j / page_size], slot j % page_size; table [batch, table_width], lens [batch]
 * (tokens that a sequence holds) and starts [batch + 1] (where its new tokens begin among `tokens` of them, ascending)
 * are int32 in device memory. In 8 bits a row of d values has the scale 2^s, s the least integer (within +-126) with
 * max|x| <= 448 * 2^s over its finite values (0 for a row of zeros), held as s + 127; its codes are x / 2^s rounded to
 * the nearest e4m3, values that are not finite NaN. In 4 bits (SAM_HIP_E2M1; d % 32 == 0) the pools are
 * [pages, kv_heads, page_size, d / 2] bytes, the scales [pages, kv_heads, page_size, d / 32], a row as sam_hip_mx_pack holds it
 * (sam_hip_mx.h): each block of 32 values with its own scale, NaN throughout if one of them is not finite.
 *
 * sam_hip_kv_write stores the new tokens' rows k, v [tokens, kv_heads, d] (strides (token, head), multiples of 16
 * bytes; NULL = contiguous): token t of sequence b goes to position lens[b] - (starts[b+1] - t), the sequence's last
 * ones. sam_hip_kv_read writes rows 0 .. max_len of every sequence to k, v [batch, max_len, kv_heads, d] of `dtype`, zeros
 * from lens[b] on (from an e4m3 or e2m1 cache in any dtype, each value rounded to it once).
 *
 * What the tables say is checked on the device. A sequence holds its keys below both lens[b] and table_width * page_size;
 * its new tokens are those of 0 .. tokens - 1 that starts names, at the positions that lens[b] and starts[b+1] as they are
 * give them, in kv-write and in attention alike. Tokens outside every sequence, at a negative position or past the table
 * are not written; a table entry outside 0 .. pages - 1 stands for a page that is not there (not written, read as zeros,
 * its keys not attended). Two positions that share a page slot must not be written in one call. Limits: d % 8 == 0, d <= 256, table_width * page_size < 2^30, fewer than 2^31 rows in
 * a pool and 2^27 in a write or a read.
 */
#define SAM_HIP_E4M3 3
#define SAM_HIP_E2M1 4
int sam_hip_kv_write(const void* k, const void* v, void* k_pages, void* v_pages, unsigned char* k_scale,
                     unsigned char* v_scale, const int* table, const int* starts, const int* lens, int dtype,
                     int cache_dtype, int tokens, int batch, int pages, int kv_heads, int page_size, int d,
                     int table_width, const long* strides_k, const long* strides_v, void* stream);
int sam_hip_kv_read(void* k, void* v, const void* k_pages, const void* v_pages, const unsigned char* k_scale,
                    const unsigned char* v_scale, const int* table, const int* lens, int dtype, int cache_dtype,
                    int batch, int max_len, int pages, int kv_heads, int page_size, int d, int table_width,
                    void* stream);

/*
 * Attention of each sequence's new tokens over its pages, the new tokens' own keys (written before) among them:
 *   out[t, hq, :] = softmax_j(scale * q[t, hq, :] . k_j) . v_j over the keys j < lens[b] of key head hq / (heads / kv_heads)
 * and, with causal, j <= t's own position lens[b] - (starts[b+1] - t). q and out [tokens, heads, d] (strides (token,
 * head), multiples of 16 bytes, out's rows apart; NULL = contiguous). A row that sees no key is 0; a key, or a value that
 * is not finite, reaches the rows that see it alone (an infinite value may come out as NaN there). Rows of no sequence
 * stay as they are, or become 0 with zero_rest. out may be q with the same strides; it must not overlap q otherwise, nor
 * the other tensors.
 * max_q and max_len are the longest chunk and the longest sequence as the caller expects them: they size the grid and
 * the key splits, and a call whose sequences exceed them is computed all the same, more slowly.
 * Workspace: sam_hip_paged_attention_workspace_size() bytes of device memory for the key splits' partial results (it
 * depends on the current device's CU count; 0 needs none, -1 is an error); calls that may overlap need their own, and
 * so does each captured graph that may run beside another. Softmax statistics and sums are f32. An e4m3 or e2m1 row is read as
 * sam_hip_kv_read would return it in q's dtype. Limits as above; heads % kv_heads == 0; scale >= 0.
 */
long sam_hip_paged_attention_workspace_size(int dtype, int cache_dtype, int tokens, int batch, int heads, int kv_heads,
                                            int d, int max_q, int max_len);
int sam_hip_paged_attention(const void* q, const void* k_pages, const void* v_pages, const unsigned char* k_scale,
                            const unsigned char* v_scale, const int* table, const int* starts, const int* lens,
                            void* out, int dtype, int cache_dtype, int tokens, int batch, int heads, int pages,
                            int kv_heads, int page_size, int d, int table_width, const long* strides_q,
                            const long* strides_o, float scale, int causal, int zero_rest, int max_q, int max_len,
                            void* workspace, long workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
