/* qe_paged.h -- C ABI of the paged key-value cache on MI355X (gfx950): gated decode attention over
 * pages (dense, or with a sliding window and first tokens that stay visible), the norm + RoPE that
 * writes them, and the operations on pages. The reference has one contiguous cache and no
 * counterpart (python/qengine/engine.py:419).
 *
 * Conventions of qe_attn.h: device pointers, strides in elements, everything enqueued on `stream`,
 * no allocation and no host sync (calls can be captured in a hipGraph), hipErrorInvalidValue before
 * any launch for arguments outside the ranges below, otherwise the launch error.
 *
 * Data:
 *   kp, vp    pools of N pages, [N][Hkv][P][256] (bf16, or E4M3FN codes with one scale per pool);
 *             P a power of two, 16 <= P <= 32768; 16-byte aligned
 *   table     int32 [B][M], rows ldt entries apart: the page that holds positions [jP, (j+1)P) of
 *             sequence b. An entry outside [0, N) names no page (-1 by convention)
 *   ref       int32 [N]: table entries that name the page. 0: the page is free
 *   pos       int32 [B]: the position of a sequence's first row. Negative: the sequence is idle: no op
 *             writes anything for it, and what its rows hold is of no account. The rows have to be
 *             there all the same: they are loaded before the position is known
 *   rows      row b * R + t of a call is the token of sequence b at position pos[b] + t
 * M * P <= 2^23 - 64 positions per sequence; 1 <= B <= 1024.
 * Every device index (pages, sequences, positions) is checked against these sizes on the device;
 * what lies outside is neither read nor written.
 */
#ifndef QE_PAGED_H
#define QE_PAGED_H

#include <stddef.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QE_PAGED_MAX_SEQS 1024

/* Gated attention of R (1..8) new rows per sequence over its pages. Row at position p attends the
 * positions j < min(p + 1, M * P) whose page is mapped and, with window > 0, for which j < sinks or
 * j >= p + 1 - window. out = bf16(softmax(q.k * scale) . v * sigmoid(gate)), rounded once, the gate
 * being qg[row][h][256:512]; a row that attends nothing is 0. Key and value rows that a row does not
 * attend do not reach it, whatever they hold (NaN, infinities). A dim of V in which a row attends +inf, -inf,
 * or both or a NaN, is +inf, -inf, or NaN before the gate, whatever the weights of those positions. A row whose
 * attended scores all are -inf, or of which one is NaN or +inf, is NaN. Sums are in fp32: finite values of V
 * beyond 2^120 / (positions attended) may overflow.
 * Two launches: partials of slices of the cache, merged by the second. A row's slices depend on its own
 * position, on B, Hkv, M * P, NS, window and sinks, and on the device's compute units, so that a row's bits
 * are the same whatever R is and whichever other rows and sequences the call holds.
 * q rows are contiguous ([B*R][Hq*256], 16-byte aligned), qg rows ldp apart, out rows ldo apart;
 * part_o fp32 [>= B*R*Hq*NS*256] (16-byte aligned) and part_ml fp32 [>= B*R*Hq*NS*2] are the
 * caller's scratch (in an order of the kernels' own): calls that may overlap need a pair each. NS >= 1, with a window NS >= 4;
 * 0 <= window < 2^23, sinks >= 0 (ignored without a window). */
hipError_t qe_attn_decode_paged(const void* q, const void* kp, const void* vp, const int* table,
                                long ldt, const int* pos, const void* qg, long ldp, float* part_o,
                                float* part_ml, void* out, long ldo, int B, int R, int Hq, int Hkv,
                                int N, int P, int M, int NS, int window, int sinks, float scale,
                                hipStream_t stream);
/* The same over pools of E4M3FN codes: a code c stands for c * k_scale (c * v_scale). */
hipError_t qe_attn_decode_paged_fp8(const void* q, const void* kp, const void* vp, const int* table,
                                    long ldt, const int* pos, const void* qg, long ldp,
                                    float* part_o, float* part_ml, void* out, long ldo, int B, int R,
                                    int Hq, int Hkv, int N, int P, int M, int NS, int window,
                                    int sinks, float scale, float k_scale, float v_scale,
                                    hipStream_t stream);

/* Norm and RoPE of the new rows, written to the pages: RMSNorm1p of q and k (eps, weights qnw / knw),
 * partial rotate-half RoPE on the first rd = 2*len(inv_freq) dims at angle pos * inv_freq (fp64), in fp32
 * and rounded once (qe_attn_prep keeps the reference's rounding after every op). q to q_out
 * ([B*R][Hq*256] contiguous), k and v to row p % P of page table[b][p / P] where 0 <= p < M * P and the page
 * is mapped. qg / k / v rows are ldp apart. Any R >= 1, B * R <= 65535 (a prompt: B = 1). Two sequences
 * that share a page must not write it in one call. */
hipError_t qe_attn_prep_paged(const void* qg, const void* k, const void* v, long ldp, const void* qnw,
                              const void* knw, const float* inv_freq, const int* pos, void* q_out,
                              void* kp, void* vp, const int* table, long ldt, int B, int R, int Hq,
                              int Hkv, int N, int P, int M, int rd, float eps, hipStream_t stream);
/* The same into pools of E4M3FN codes: the code nearest to x * (1 / scale), saturated at +-448. */
hipError_t qe_attn_prep_paged_fp8(const void* qg, const void* k, const void* v, long ldp,
                                  const void* qnw, const void* knw, const float* inv_freq,
                                  const int* pos, void* q_out, void* kp, void* vp, const int* table,
                                  long ldt, int B, int R, int Hq, int Hkv, int N, int P, int M, int rd,
                                  float eps, float k_scale, float v_scale, hipStream_t stream);

/* ---- operations on pages. `table` and `ref` are the allocation: ref[i] is the number of table entries
 * that name page i. Everything is decided on the device, in one order whatever the timing: where ids are
 * given out, the lowest free ones, in the order of sequences (or pairs) and then of positions. Calls on one
 * allocation must follow one another (one stream, or ordered ones). 1 <= N <= 2^24.
 * `missing` (int32 [1]) is written by every call that takes it: the pages it could not give. */

/* Releases every page of sequence b whose positions all lie in [first[b], last[b]): ref - 1, entry -1.
 * A finished sequence: [0, INT_MAX); the pages behind a window: [sinks, p + 1 - window); a truncation to n
 * positions: [n, INT_MAX). */
hipError_t qe_kv_pages_free(int* table, long ldt, int* ref, const int* first, const int* last, int B,
                            int M, int N, int P, hipStream_t stream);
/* Maps the pages that positions [pos[b], pos[b] + count[b]) need and that are not mapped yet. missing[0]:
 * those for which no page was free, or that lie past the table's width. */
hipError_t qe_kv_pages_extend(int* table, long ldt, int* ref, const int* pos, const int* count,
                              int* missing, int B, int M, int N, int P, hipStream_t stream);
/* Bytes of workspace of fork and compact (int32 [2 N + 8]). */
size_t qe_kv_pages_ws_size(int N);
/* Sequence dst[i] becomes a copy of the first length[i] positions of sequence src[i], for m pairs: dst's own
 * pages are released, pages wholly below the length are shared (ref + 1), a last partial page is copied
 * into a page of its own. Pages that src does not have, dst does not get. A pair is refused (it changes
 * nothing and counts in missing) if src or dst is not a sequence of the table, or dst is also a source or
 * the dst of another pair. missing[0]: partial pages for which none was free, plus refused pairs.
 * Neither sequence may write below length afterwards (its pages there are shared): to go back further, fork to
 * the earlier length.
 * kp / vp: `layers` pools of N pages of page_bytes (a multiple of 16) each, one after another.
 * 1 <= m <= 1024. */
hipError_t qe_kv_pages_fork(int* table, long ldt, int* ref, const int* src, const int* dst,
                            const int* length, int m, void* kp, void* vp, int layers, size_t page_bytes,
                            int* missing, void* ws, int B, int M, int N, int P, hipStream_t stream);
/* Moves pages so that the U pages in use are pages 0 .. U - 1: the k-th page in use with id >= U goes to the
 * k-th free id < U. Table, ref and data follow. */
hipError_t qe_kv_pages_compact(int* table, long ldt, int* ref, void* kp, void* vp, int layers,
                               size_t page_bytes, void* ws, int B, int M, int N, hipStream_t stream);
/* Copies the data of page src[i] to page dst[i] in every layer of both pools, for m pairs. A pair is left out
 * if an id lies outside [0, N), if src[i] == dst[i], if a later pair has the same dst, or if dst[i] is any
 * pair's source: what is copied does not depend on an order. 1 <= m <= 65535. */
hipError_t qe_kv_pages_copy(void* kp, void* vp, int layers, size_t page_bytes, const int* src,
                            const int* dst, int m, int N, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* QE_PAGED_H */
