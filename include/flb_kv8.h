/*
 * flb_kv8.h — C ABI of the 8-bit K/V cache of the B200 (sm_100a) attention path: tokens are appended in 8 bits with
 * one scale per block of rows and K/V head, single-token attention reads the codes, and rows that drew little
 * attention are evicted.  It stands beside the fp32/fp16 cache of flb_attn.h and follows its manners: plain C, device
 * pointers, sizes as ints / size_t, the stream a cudaStream_t passed as void*; the library allocates nothing, never
 * synchronises, never exits and never throws; every entry point returns a flb_status.  Calls that can run at the same
 * time need scratch of their own.  The reference has no counterpart (its cache is fp32, open_decoder.h:72-77).
 */
#ifndef FLB_KV8_H
#define FLB_KV8_H

#include "flb_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* What a code stands for: value = scale * int8, or scale * e4m3. */
typedef enum flb_kv8_code {
    FLB_KV8_I8 = 0,
    FLB_KV8_E4M3 = 1
} flb_kv8_code;

/* The cache of one layer.  Row r of sequence b and K/V head h: codes [b][h][r][0..d), scale [b][h][r / block_len].
 * Rows at or behind a sequence's length may hold anything.
 *
 * How rows get in (append, decode and evict alike): per block and head, K and V apart, amax = the largest magnitude of
 * the rows that come in, need = amax / top (top = 127 for int8, 448 for e4m3), and
 *     scale' = need               for a block whose first row is new,
 *     scale' = max(scale, need)   for a block that holds rows already (an eviction fills holes, so always this); if it grew,
 *                                 the codes it held become rne(code * (scale / scale')),
 *     new code = rne(x / scale')  (0 where scale' is 0 or not finite; held to -top..top, which matters for subnormal scales),
 * each operation one IEEE fp32 operation, so two calls that store the same rows store the same bits.  A block
 * into which an infinity or NaN was stored has an infinite or NaN scale from then on: its rows read as NaN. */
typedef struct flb_kv8_cache {
    int batch_size;    /* B                                                             */
    int kv_head_num;   /* Hkv                                                           */
    int size_per_head; /* d: 64, 128 or 256                                             */
    int total_len;     /* T, row capacity of one (b, h) slab; a multiple of block_len   */
    int block_len;     /* rows that share a scale: 16, 32, 64 or 128                    */
    int code_type;     /* flb_kv8_code                                                  */
    void *k_codes;     /* [B,Hkv,T,d], one byte each                                    */
    void *v_codes;
    float *k_scale;    /* [B,Hkv,T/block_len]                                           */
    float *v_scale;
    int *row_pos;      /* [B,Hkv,T] position of every row in its text; NULL = row number.
                          Needed once rows have been evicted and a distance bias or key_begin is used */
} flb_kv8_cache;

/* Appends seq_len tokens (1 or more) behind the rows that are there.  Accumulated attention (weight_in, weight_out below) is the caller's: what stands in
 * its buffer for the new rows, left from rows that an eviction dropped for instance, is to be zeroed before the next decode. */
typedef struct flb_kv8_append_params {
    flb_kv8_cache cache;
    int seq_len;            /* S                                                        */
    int start_pos;          /* rows already in the cache, when past_lens is NULL        */
    const int *past_lens;   /* device int[B] or NULL                                    */
    const int *new_lens;    /* device int[B] or NULL: tokens of sequence b that count (0..S; the rest of a padded
                               batch is not stored); NULL = S                            */
    const int *token_pos;   /* device int[B] or NULL: position of the first new token; NULL = the cached rows.  Positions that pass
                               INT_MAX are kept as INT_MAX in row_pos                     */
    int input_mode;         /* flb_input_mode                                           */
    const void *k;          /* [B,S,Hkv,d]                                              */
    const void *v;
    int kv_row_stride;      /* elements between the rows of two tokens; 0 = Hkv * d     */
    const float *act_scale; /* FLB_IN_INT32: [B*S]                                      */
    const float *k_w_scale; /* FLB_IN_INT32: [Hkv*d]                                    */
    const float *v_w_scale;
    const float *freq_cis;  /* RoPE table as in flb_attn.h, row = position; NULL = none */
    int freq_rows;          /* rows of the table                                        */
    unsigned *status;       /* device word, error bits are OR-ed in; may be NULL        */
} flb_kv8_append_params;

/* One new token per sequence: appended as above, then attended over with everything cached.
 *   x[r]  = softmax_scale * q . k[r];  softcap > 0: x = softcap * tanh(x / softcap);
 *   slope: x -= alibi_slopes[h] * |token position - position of row r|
 * over the rows 0..past whose position is >= key_begin[b]; no such row gives a zero output row.
 * q head h reads K/V head h / (head_num / kv_head_num). */
typedef struct flb_kv8_decode_params {
    flb_kv8_cache cache;
    int head_num;            /* H, a multiple of kv_head_num                            */
    int start_pos;           /* rows already in the cache, when past_lens is NULL       */
    const int *past_lens;    /* device int[B] or NULL                                   */
    int max_past_len;        /* host's upper bound on past_lens (0 = total_len - 1); sizes the grid */
    const int *token_pos;    /* device int[B] or NULL: position of the new token; NULL = the cached rows */
    int input_mode;          /* flb_input_mode                                          */
    const void *q;           /* [B,1,H,d]                                               */
    const void *k;           /* [B,1,Hkv,d]                                             */
    const void *v;
    int q_row_stride;        /* elements between two sequences' rows; 0 = H * d         */
    int kv_row_stride;       /* 0 = Hkv * d                                             */
    const float *act_scale;  /* FLB_IN_INT32: [B]                                       */
    const float *q_w_scale;  /* FLB_IN_INT32: [H*d], [Hkv*d], [Hkv*d]                   */
    const float *k_w_scale;
    const float *v_w_scale;
    const float *freq_cis;
    int freq_rows;
    float softmax_scale;
    float softcap;             /* 0 = none, else 2^-10 .. 2^40                          */
    const float *alibi_slopes; /* [H] or NULL                                           */
    const int *key_begin;      /* device int[B] or NULL                                 */
    /* Accumulated attention, for flb_kv8_evict(): weight_out[b][h][r] = weight_in[b][h][r] + the sum of the weights that
     * the group's q heads give row r, for r = 0..past (row past starts from 0); further rows are left alone.  Both
     * [B,Hkv,T], 16-byte aligned; they may be the same buffer.  NULL, NULL = off. */
    const float *weight_in;
    float *weight_out;
    void *out;               /* [B,H,1,d]                                               */
    int out_dtype;           /* flb_dtype                                               */
    void *scratch;           /* flb_kv8_decode_workspace_bytes()                        */
    size_t scratch_bytes;
    int scratch_zeroed;      /* promise: the first flb_kv8_counter_bytes() bytes are zero on entry.  They are left zero; a call of
                                other sizes in between may write there */
    int split_len;           /* rows of one split of a sequence, a multiple of 128 up to 2048; 0 = default, by total_len.  Results
                                depend on it and on each sequence alone, never on the batch or the grid.  Where total_len is far
                                above the lengths in use, name that of a slab of those (512 up to 8192 rows) */
} flb_kv8_decode_params;

/* Cuts every sequence down to `budget` rows per head.  Of the n cached rows, those at a position below `sinks` or at or
 * behind next_pos[b] - recent come first, the others follow by falling weight (NaN counts as the largest), ties to the
 * lower row; the first m = min(n, budget) are kept.  Kept rows below m stay where they are; the i-th hole below m takes the i-th
 * kept row at or behind m (codes are brought to the block's scale by the rule above), so only those rows move and the order of
 * rows is no longer that of positions: row_pos says where each belongs.  Weights and positions go along, to weight_out and pos_out,
 * which may be weight and cache.row_pos themselves. */
typedef struct flb_kv8_evict_params {
    flb_kv8_cache cache;     /* row_pos is needed                                       */
    int start_pos;           /* cached rows n, when past_lens is NULL                   */
    const int *past_lens;    /* device int[B] or NULL; 0..total_len                     */
    int *len_out;            /* device int[B]: m; may be past_lens                      */
    int budget;              /* rows to keep, >= 1                                      */
    int recent;              /* sinks + recent <= budget                                */
    int sinks;
    const int *next_pos;     /* device int[B]: position of the next token; needed when recent > 0 */
    const float *weight;     /* [B,Hkv,T]; this, the two results and row_pos 16-byte aligned */
    float *weight_out;       /* [B,Hkv,T], rows 0..m-1 are written                      */
    int *pos_out;
    void *scratch;           /* flb_kv8_evict_workspace_bytes(); need not be zeroed     */
    size_t scratch_bytes;
} flb_kv8_evict_params;

/* Error bits in the status word (the head of the decode and evict scratch, *status of an append). */
#define FLB_KV8_STATUS_BAD_LEN 4u   /* a cached length, or length + tokens, outside the slab or above max_past_len: that sequence
                                       was left alone, and its output rows are zero */
#define FLB_KV8_STATUS_BAD_POS 32u  /* a position outside the RoPE table: the nearest row was used */

/* Host-side argument checks only (no CUDA call); the launch entry points run them first.  Beside what the fields say, a call is refused with
 * FLB_ERR_TOO_LARGE where batch_size * head_num passes 2^24, a row of heads 2^31 elements, or a grid its limits (an append, or a decode of more than 8
 * (d = 256: 4) q heads per K/V head: more than 65535 sequences, or blocks that one call can touch). */
int flb_kv8_validate_append(const flb_kv8_append_params *p);
int flb_kv8_validate_decode(const flb_kv8_decode_params *p);
int flb_kv8_validate_evict(const flb_kv8_evict_params *p);

/* Scratch of a decode call on a full cache of these sizes (cache sizes, head_num, split_len, and whether weight_out is
 * set are read), the bytes at its start that have to be zero, and the scratch of an eviction. */
int flb_kv8_decode_workspace_bytes(const flb_kv8_decode_params *p, size_t *bytes_out);
int flb_kv8_counter_bytes(const flb_kv8_decode_params *p, size_t *bytes_out);
int flb_kv8_evict_workspace_bytes(const flb_kv8_evict_params *p, size_t *bytes_out);

int flb_kv8_append(const flb_kv8_append_params *p, void *cuda_stream);
int flb_kv8_decode(const flb_kv8_decode_params *p, void *cuda_stream);
int flb_kv8_evict(const flb_kv8_evict_params *p, void *cuda_stream);

#ifdef __cplusplus
}
#endif
#endif /* FLB_KV8_H */
