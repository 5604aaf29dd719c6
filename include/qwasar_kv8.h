/* qwasar_kv8.h -- the 8-bit K/V cache of the B200 backend: append, read, attention over it, and the
 * rotary positions that go in front of it.
 *
 * An extension of qwasar_cuda.h with the same handles, command buffers, alignment rules and errors:
 * an op given arguments it does not take returns false and encodes nothing, and qw_cmd_error says why.
 * Operands must live on the device of the command buffer.  Plain C99. */
#ifndef QWASAR_KV8_H
#define QWASAR_KV8_H

#include "qwasar_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions in both layouts ----------------------------------------
 * Beside qw_op_rope_partial (f32, in place, half layout, three position axes): either layout, f32 or
 * bf16, rows apart by a stride, in place or into another buffer, frequencies scaled for long contexts.
 * Pair j < rotary_dim / 2 of every head of row r turns by a = pos[r] * inv_freq[j]:
 *   (x1, x2) -> amp * (x1 cos a - x2 sin a, x2 cos a + x1 sin a)
 * QW_ROPE_HALF: x1, x2 = elements j and j + rotary_dim / 2; QW_ROPE_INTERLEAVED: 2j and 2j + 1.  Dims
 * from rotary_dim on are copied.  The angle is formed and reduced in 64 bits: positions may be any
 * int32.  pos int32 [rows], inv_freq f32 [rotary_dim / 2]; x and y are rows of heads * head_dim
 * elements, x_stride and y_stride elements apart (a slice of a joint projection's rows is fine).  y may
 * be x with the same stride; other overlaps, head_dim over 4096, an odd rotary_dim and strides below
 * the row's width are refused (false, and qw_cmd_error says why).  rows 0 is nothing to do: true. */
typedef enum { QW_ROPE_HALF = 0, QW_ROPE_INTERLEAVED = 1 } qw_rope_layout;
bool qw_op_rope(qw_cmd c, qw_ref y, qw_ref x, qw_ref pos, qw_ref inv_freq, int32_t rows, int32_t heads,
                int32_t head_dim, int32_t rotary_dim, qw_rope_layout layout, int64_t y_stride,
                int64_t x_stride, float amp, qw_dtype io);
/* inv_freq [rotary_dim / 2] and amp (may be NULL) for contexts `factor` times the original one.
 * PLAIN: theta^(-2j / rotary_dim).  LINEAR: that over factor.  NTK: theta grown by
 * factor^(rotary_dim / (rotary_dim - 2)), so that the slowest pair is stretched by factor and the
 * fastest kept.  BANDS: pairs that turn more than beta_fast times over original_ctx are kept, those
 * below beta_slow divided by factor, a linear ramp over j in between; amp = 0.1 ln(factor) + 1 (the
 * other kinds: 1).  Host arithmetic in 64 bits, no device needed.  False on arguments that do not make
 * sense (theta or factor not positive, BANDS without 0 < beta_slow < beta_fast, theta > 1 and factor >= 1). */
typedef enum { QW_ROPE_PLAIN = 0, QW_ROPE_LINEAR = 1, QW_ROPE_NTK = 2, QW_ROPE_BANDS = 3 } qw_rope_scaling;
bool qw_rope_scaled_tables(float *inv_freq, float *amp, int32_t rotary_dim, float theta, qw_rope_scaling kind,
                           float factor, int32_t original_ctx, float beta_fast, float beta_slow);

/* ---- the 8-bit K/V cache --------------------------------------------------------
 * Half the bytes of the bf16 cache: an element is an e4m3 code times 2^e, one e per 64 tokens of one
 * head, the smallest whole number in [-60, 119] with largest magnitude <= 448 * 2^e; its byte is e + 127
 * (bytes outside that range read as the nearest).  One layer of a plain cache buffer is
 *   codes uint8 [kv_heads, max_ctx, 256] | exponents uint8 [kv_heads, ceil(max_ctx / 64)] | padding
 * = qw_kv8_layer_bytes(kv_heads, max_ctx, 256) bytes, layers one after the other, the buffer on a
 * 128-byte boundary.  Or an arena: pages of 128 tokens mapped as tokens arrive, from a pool that bf16
 * and 8-bit arenas may share; its layers are addressed at the same offsets, layer * qw_kv8_layer_bytes.
 * qw_buf_free, qw_kv_arena_trim, _pages_in_use and _bytes_committed work on both kinds of arena; ops
 * given the other kind refuse it. */
size_t  qw_kv8_layer_bytes(int32_t kv_heads, int32_t max_ctx, int32_t head_dim);   /* 0 on bad arguments */
qw_buf  qw_kv8_arena_alloc(int32_t n_layers, int32_t kv_heads, int32_t max_ctx, int32_t head_dim, uint32_t shuffle_seed);
qw_buf  qw_kv8_arena_alloc_in(qw_buf pool, int32_t n_layers, int32_t kv_heads, int32_t max_ctx, int32_t head_dim);
/* Appends rows of K and V (f32 or bf16, each row kv_heads * 256 elements, row_stride elements apart, a
 * multiple of 16 bytes) at base_pos, like qw_op_kv_write.  A block that begins with this call takes its
 * exponent from the call's rows; one that holds rows already keeps its exponent, or moves to a larger
 * one and its codes with it.  A rewind needs nothing: rows past the new end are overwritten, and the
 * exponent of the block that is cut only stays larger than it would have to be.  An append ends the
 * cache: rows behind it do not follow when its block's exponent moves.  A NaN is stored as
 * zero and an infinity as the block's largest code; either is reported by qw_cmd_error after
 * qw_cmd_wait.  The batch form takes n_seq sequences of `rows` rows each in one launch per 64.  A cache
 * may appear only once in a call.  An append inside a graph capture needs its pages mapped before. */
bool    qw_op_kv8_write(qw_cmd c, qw_ref kcache, qw_ref vcache, qw_ref k, qw_ref v, int32_t rows, int32_t kv_heads,
                        int32_t head_dim, int32_t max_ctx, int32_t base_pos, int64_t row_stride, qw_dtype io);
bool    qw_op_kv8_write_batch(qw_cmd c, int32_t n_seq, const qw_ref *kcache, const qw_ref *vcache, const qw_ref *k,
                              const qw_ref *v, const int32_t *base_pos, int32_t rows, int32_t kv_heads,
                              int32_t head_dim, int32_t max_ctx, int64_t row_stride, qw_dtype io);
/* dst [kv_heads, n, 256] (f32 or bf16; both hold the values exactly) = positions [pos0, pos0 + n) of one
 * layer's K or V.  Pages of an arena that were never mapped read as zeros. */
bool    qw_op_kv8_read(qw_cmd c, qw_ref dst, qw_ref cache, int32_t pos0, int32_t n, int32_t kv_heads, int32_t head_dim,
                       int32_t max_ctx, qw_dtype io);
/* Causal attention over an 8-bit cache, like qw_op_attn: row r of query head h attends positions
 * [0, base_pos + r] of kv head h / (q_heads / kv_heads).  q, out [rows, q_heads, 256], f32 or bf16; gate
 * a null ref, or element (r, h, d) at gate[(r*q_heads + h)*gate_stride + d], in the same type: out is
 * multiplied by its sigmoid.  f32 is carried through (operands as two fp16 parts, sums in f32: about
 * 1e-6); bf16 rounds the softmax weights to fp16.  Up to 32 query rows per kv head (rows * grouping) run
 * as one split-KV launch for up to 64 sequences; more of them, in bf16, as a tcgen05 launch per sequence or
 * in chunks of the former, whichever should take less time; in f32 in chunks.  Grouping at most 32.
 * Positions from base_pos + rows on may hold anything; a NaN code among the visible ones (qw_op_kv8_write
 * stores none) makes the rows that see it NaN.  Query rows count as finite up to 2^100.  K and V may lie in
 * caches of different kinds; sequences of a batch may share a cache, outputs may not.  Partial sums live in
 * scratch of the command buffer: calls on one command buffer follow one another, two that may run at once
 * (two streams, two captured graphs) need two command buffers, which live as long as the graphs captured on
 * them. */
bool    qw_op_attn_kv8(qw_cmd c, qw_ref out, qw_ref gate, qw_ref q, qw_ref kcache, qw_ref vcache, int32_t rows,
                       int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_ctx, int32_t base_pos,
                       float scale, int32_t gate_stride, qw_dtype io);
bool    qw_op_attn_kv8_batch(qw_cmd c, int32_t n_seq, const qw_ref *out, const qw_ref *gate, const qw_ref *q,
                             const qw_ref *kcache, const qw_ref *vcache, const int32_t *base_pos, int32_t rows,
                             int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_ctx, float scale,
                             int32_t gate_stride, qw_dtype io);

#ifdef __cplusplus
}
#endif
#endif /* QWASAR_KV8_H */
