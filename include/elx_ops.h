/*
 * C ABI of libelx_ops.so -- operators of a training step beside the 32-bit optimizer step, for gfx950 (MI355X):
 *
 *   adam8       Adam / AdamW over the tables of elx_abi.h with exp_avg and exp_avg_sq held in 8 bits
 *   layer norm  forward and backward, with the reduction of the gradients of weight and bias
 *   embedding   lookup with scaling, and the dense gradient of the table
 *
 * The conventions are those of elx_abi.h: plain C, every table pointer is a device pointer, the caller owns all
 * memory, nothing is allocated, all work goes asynchronously to the hipStream_t passed as `stream`, and every function
 * returns 0, a hipError_t (> 0) or one of the ELX_E_* codes (< 0; elx_strerror of libelx_hip.so has the texts).
 */
#ifndef ELX_OPS_H
#define ELX_OPS_H

#include "elx_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ELX_OPS_VERSION 1

int elx_ops_version(void);

/* The first 16 hex digits of the SHA-256 over the sources of this library, as the build passed it in ("" without). */
const char *elx_ops_source_sha(void);

/*
 * The 8-bit optimizer state.  A flat buffer of n elements is cut into blocks of elx_state8_block() = 256 elements; it has
 * n codes of exp_avg, n codes of exp_avg_sq and one 16-bit word per block: the exponent E of exp_avg in the low byte, the
 * one of exp_avg_sq in the high byte.
 *   exp_avg     code: sign, 4 exponent and 3 mantissa bits without infinities (torch.float8_e4m3fn);
 *               value = code * 2^(E - 135), rounded to nearest even
 *   exp_avg_sq  code: 5 exponent and 3 mantissa bits, subnormals below; 255 is NaN;
 *               value = float32(bits = code << 20) * 2^(E - 31)
 * E is the smallest exponent for which the largest finite magnitude of the block is at most 1.75 * 2^(E - 127), and for
 * E = 0, where fp32 has no implicit bit, at most 1.5 * 2^-127: (bits of the largest + 0x1FFFFF) >> 23.  The
 * scales are powers of two, so what the codes hold is exact in fp32 (and in bfloat16), and writing back what was read
 * changes no value.  (Under E = 255 a code could stand for 2^128, which fp32 does not hold: what is finite is written as
 * 1.875 * 2^127 at most.)
 * exp_avg_sq moves by (1 - beta2) of itself in a step, far less than the distance of two codes: rounded to nearest it
 * would never move.  It is rounded up or down at random with the right expectation: 20 bits r per element are added below
 * the mantissa that is kept and the sum is cut off.  The bits depend on (salt, element, step) alone, so a step gives the
 * same result however it is launched:
 *   mix(x):  x ^= x >> 16; x *= 0x6A09E667; x ^= x >> 15; x *= 0xBB67AE85; x ^= x >> 16     (32-bit, wrapping)
 *   key  = mix(block ^ mix(salt * 0x9E3779B9 + step))
 *   word = mix(key + lane * 0x9E3779B9)         lane = (element of the block) / 4
 *   r    = rotate_right(word, 8 * (element of the block mod 4)) >> 12
 * A value that is not zero never becomes zero: the next step would divide by eps alone.  exp_avg_sq is a sum of squares and
 * its code has no sign: -0.0 is zero, and of a negative value, which only a checkpoint could bring, the magnitude is held.
 * A value that is not finite becomes NaN; its neighbours in the block keep theirs.
 */
typedef struct ElxState8 {
    uint16_t *scales;      /* word of the row's first block; ElxChunk.m / .v of the row point to its first codes */
    uint32_t first_block;  /* place of that block in the whole buffer: a row starts at a block boundary */
    uint32_t salt;         /* place of the buffer among the buffers of the optimizer */
} ElxState8;

uint32_t elx_sizeof_state8(void);
uint32_t elx_state8_block(void);

/*
 * elx_adam_step_mt (elx_abi.h) over an 8-bit state: d_chunks as there, with m and v pointing to codes (4-byte aligned),
 * and one ElxState8 record per row in d_state.  The arithmetic on the values the codes stand for is that of
 * elx_adam_step_mt, the change of a master weight to within 2^-20 of itself (IEEE division and square root where eps is
 * below 2^-36); master weights and low-precision copy come from the new moments before they are rounded.  The
 * rounding of exp_avg_sq takes its step from bits 8..31 of ElxHyper.flags (the step count modulo 2^24).  Elements that no
 * segment covers keep their values (to nearest, where the exponent of their block has changed).
 *   elx_adam8_step_mt        hyper records in device memory
 *   elx_adam8_step_args_mt   1..32 hyper records in HOST memory, carried in the arguments of the launch
 *   elx_adam8_step_gated_mt  unscale parameters and skip flag from the gate words of the device records
 * Tables are checked by elx_check_tables (elx_abi.h) and elx_check_state8.  blocks_per_cu 0: the default.
 */
int elx_adam8_step_mt(const ElxChunk *d_chunks, const ElxState8 *d_state, uint32_t n_chunks, const ElxSeg *d_segs,
                      uint32_t n_segs, const ElxHyper *d_hypers, uint32_t n_hypers, uint64_t total_tiles,
                      uint32_t grid_tiles_per_chunk, float div_scale, int grad_dtype, int lowp_dtype, uint32_t flags,
                      uint32_t blocks_per_cu, void *stream);
int elx_adam8_step_args_mt(const ElxChunk *d_chunks, const ElxState8 *d_state, uint32_t n_chunks, const ElxSeg *d_segs,
                           uint32_t n_segs, const ElxHyper *h_hypers, uint32_t n_hypers, uint64_t total_tiles,
                           uint32_t grid_tiles_per_chunk, float div_scale, int grad_dtype, int lowp_dtype, uint32_t flags,
                           uint32_t blocks_per_cu, void *stream);
int elx_adam8_step_gated_mt(const ElxChunk *d_chunks, const ElxState8 *d_state, uint32_t n_chunks, const ElxSeg *d_segs,
                            uint32_t n_segs, const ElxHyper *d_hypers, uint32_t n_hypers, uint64_t total_tiles,
                            uint32_t grid_tiles_per_chunk, int grad_dtype, int lowp_dtype, uint32_t flags,
                            uint32_t blocks_per_cu, void *stream);

/* Host copies of the state rows of an update before they are uploaded: NULL, odd address, a place beyond 2^32 blocks. */
int elx_check_state8(const ElxChunk *h_chunks, const ElxState8 *h_state, uint32_t n_chunks);

/*
 * elx_state8_read   values of the elements [begin, begin + n) of a buffer, as fp32 or bf16; m_out or v_out may be NULL
 * elx_state8_write  n values (fp32) into codes and exponents of one moment (0 exp_avg, 1 exp_avg_sq) from the start of a
 *                   buffer, rounded to nearest (exp_avg_sq: halves up); the other moment's exponents are left alone
 */
int elx_state8_read(const uint8_t *m_codes, const uint8_t *v_codes, const uint16_t *scales, uint64_t begin, uint64_t n,
                    void *m_out, void *v_out, int out_dtype, void *stream);
int elx_state8_write(const float *values, uint64_t n, int moment, uint8_t *codes, uint16_t *scales, void *stream);

/*
 * Layer norm over rows of `cols` elements (1..elx_layer_norm_max_cols()), all tensors of one type (fp32, fp16, bf16):
 *   forward   y = (x - mean) / sqrt(var + eps) * w + b;  w and b may be NULL (1 and 0), mean and rstd (fp32, `rows` each;
 *             what backward needs) too.  y is packed, x has rows `x_stride` elements apart.
 *   backward  dx (packed; may be NULL), dw and db (either may be NULL).  The workspace holds one partial row of dw and
 *             db per workgroup, elx_layer_norm_bwd_workspace() bytes, and is needed only for dw or db; contents ignored.
 * A row is read once and written once.  Sums are in fp32; the order of every sum is fixed.
 */
uint32_t elx_layer_norm_max_cols(void);
uint64_t elx_layer_norm_bwd_workspace(uint64_t rows, uint32_t cols);
int elx_layer_norm_fwd(const void *x, const void *w, const void *b, void *y, float *mean, float *rstd, uint64_t rows,
                       uint32_t cols, uint64_t x_stride, float eps, int dtype, void *stream);
int elx_layer_norm_bwd(const void *dy, const void *x, const void *w, const float *mean, const float *rstd, void *dx,
                       void *dw, void *db, void *workspace, uint64_t workspace_bytes, uint64_t rows, uint32_t cols,
                       uint64_t dy_stride, uint64_t x_stride, int dtype, void *stream);

/*
 * Embedding of n tokens (1..2^26) in a table of `vocab` (1..2^30) rows of `cols` (1..2^20) elements of one type (fp32,
 * fp16, bf16); indices are 4- or 8-byte integers.
 *   forward   out[i] = scale * table[index[i]], multiplied in fp32 and rounded once.  An index outside [0, vocab) reads
 *             nothing; its row of `out` is NaN.
 *   backward  dtable[v] = scale * (sum of dy[i] over index[i] == v), summed in fp32 in a fixed order and rounded
 *             once; rows that no token names are zero.  All of dtable is written.  Tokens whose index is `padding` (< 0:
 *             none) or outside the table add nothing.  Rows of dy are `dy_stride` elements apart.  The workspace
 *             (elx_embedding_bwd_workspace() bytes, 16-byte aligned, contents ignored) holds the sorted tokens and partial sums.
 *             n * cols and vocab * cols are at most 2^34.
 */
int elx_embedding_fwd(const void *index, int index_bytes, uint64_t n, const void *table, uint64_t vocab, uint32_t cols,
                      float scale, void *out, int dtype, void *stream);
uint64_t elx_embedding_bwd_workspace(uint64_t n, uint64_t vocab, uint32_t cols);
int elx_embedding_bwd(const void *index, int index_bytes, uint64_t n, const void *dy, uint64_t dy_stride, void *dtable,
                      uint64_t vocab, uint32_t cols, float scale, int64_t padding, void *workspace,
                      uint64_t workspace_bytes, int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ELX_OPS_H */
