/*
 * C ABI of libmkb200_sequences.so: what happens to sequences between two decoding steps, for the caches and
 * states of libmkb200.so and libmkb200_hybrid.so.  No counterpart in the reference, which decodes greedily with a
 * cache that only grows (megakernels/generators.py:121-163).
 *
 *   mkb_beam_select    beam search: the best continuations of every group of beams, from a step's logits
 *   mkb_reorder_slots  every slot takes another slot's cache rows or state, all at once and in place
 *   mkb_key_weights    the softmax weight that a run of queries gives each cached key, accumulated
 *   mkb_select_rows    which rows of a cache stay: the first, the last, and the heaviest of the others
 *   mkb_move_rows      moves those rows to the front of the caches, in place
 *
 * Plain pointers and sizes; all pointers are device memory of the current device, owned by the caller.  Every entry
 * is asynchronous on the given stream (a cudaStream_t; NULL is the legacy default stream), allocates nothing and may be
 * captured into a graph.  Workspaces need no initial contents; two calls that may overlap on the GPU (other streams,
 * two graphs) need two.  Nothing is launched when a check fails.
 */
#ifndef MKB200_SEQUENCES_H
#define MKB200_SEQUENCES_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MKBS_ABI_VERSION 1

enum MkbsCode { /* same values as MkbCode of mkb200.h */
    MKBS_OK = 0,
    MKBS_ERR_INVALID_ARGUMENT = 1,
    MKBS_ERR_CUDA = 2,
    MKBS_ERR_DEVICE_TIMEOUT = 3,
    MKBS_ERR_UNSUPPORTED = 5
};

enum MkbsDtype { MKBS_BF16 = 0, MKBS_F32 = 1 };

/*
 * The `k` best of a group's beams * vocab continuations, best first.  Continuation (b, v) has the score
 * scores[b] + log softmax(logits[b])[v]; equal scores go to the lowest (b, v).  A beam that is done has one
 * continuation, `eos` at scores[b].  Scores are compared in 64 bits; the sum of exponentials is fp32 over runs of the vocabulary
 * and fp64 over the runs.
 *
 * A logit that is minus infinity or not a number is a continuation of score minus infinity; so are all of a beam whose
 * score is not finite, or whose logits are all minus infinity.  They are taken, lowest (b, v) first, where there are no others.
 * Logits of plus infinity share their beam's whole probability.  Outputs are not in the place of inputs.
 */
typedef struct MkbsBeams {
    uint32_t struct_bytes;
    int32_t dtype;             /* MkbsDtype of the logits */
    int32_t groups, beams, vocab;
    int32_t k;                 /* 1..MKBS_MAX_BEST, at most beams * vocab */
    int64_t row_stride;        /* elements from one beam's logits to the next's, at least vocab; any alignment */
    const void *logits;        /* [groups * beams, vocab] */
    const float *scores;       /* [groups, beams] or NULL: zero */
    const uint8_t *done;       /* [groups, beams] or NULL: none is */
    int32_t eos;               /* -1: no token ends a beam (then `done` must be NULL) */
    int32_t reserved;
    float *out_scores;         /* [groups, k] */
    int32_t *out_parents;      /* [groups, k]: row of the logits, group * beams + beam */
    int32_t *out_tokens;       /* [groups, k] */
    uint8_t *out_done;         /* [groups, k] or NULL: the token is eos, or the beam was done */
    void *workspace;           /* mkb_beam_bytes, 16-byte aligned */
    size_t workspace_bytes;
} MkbsBeams;
#define MKBS_MAX_BEAMS 64      /* per group */
#define MKBS_MAX_BEST 128
#define MKBS_MAX_BEAM_WORK (1 << 30) /* beams * vocab * k */
size_t mkb_beam_bytes(const MkbsBeams *b); /* 0: not valid */
int mkb_beam_select(const MkbsBeams *b, void *cuda_stream);

/*
 * x[slot] <- x[parents[slot]] for all slots at once, in place, for every region.  Of a slot's rows those from `first` on that its
 * parent holds move (rows below `first` are alike in a slot and its parent: a shared prompt); what lies behind
 * lengths[parent] stays as it was.  A parent outside 0..slots-1 leaves its slot as it is.  Regions share no bytes.
 */
typedef struct MkbsRegion {
    void *base;
    int32_t outer;             /* layers */
    int32_t rows;              /* per slot and layer */
    int64_t outer_stride, slot_stride; /* bytes */
    int64_t row_bytes;         /* rows of a slot lie one behind the other */
} MkbsRegion;
#define MKBS_MAX_REGIONS 48    /* per call */
#define MKBS_MAX_SLOTS 256
typedef struct MkbsReorder {
    uint32_t struct_bytes;
    int32_t slots;
    int32_t num_regions;
    int32_t first;
    const MkbsRegion *regions; /* host */
    const int32_t *parents;    /* [slots] */
    const int32_t *lengths;    /* [slots]: rows that a slot holds (above a region's rows: all); NULL: all */
    int32_t *status;           /* 16 words that a wait for the call's own copies which gives up (2 s; not all rows have moved then) writes to (code, block), or NULL: not recorded */
} MkbsReorder;
int mkb_reorder_slots(const MkbsReorder *r, void *cuda_stream);

/*
 * weights[layer][sequence][head][j] += the softmax weights that the queries give key j of this key/value head, summed over the
 * queries and over the heads / kv_heads query heads that share it.  The queries of a sequence are those of its last
 * rows: with n rows query t sees the rows up to n - queries + t (none of them where that is negative).  Products are bf16,
 * everything else is fp32; a key's sum has a fixed order.  Weights behind a sequence's rows stay as they are.
 */
typedef struct MkbsKeyWeights {
    uint32_t struct_bytes;
    int32_t layers, sequences, queries;
    int32_t heads, kv_heads;   /* at most 128 query heads per key/value head */
    int32_t dim;               /* 64 or 128 */
    int32_t positions;         /* rows of a sequence's cache */
    int32_t length;            /* rows that every sequence holds, where `lengths` is NULL */
    float scale;
    const int32_t *lengths;    /* [sequences] or NULL; below 0 counts as 0, above `positions` as that */
    const void *q;             /* bf16 [layers, sequences, queries, heads * dim], 16-byte aligned */
    int64_t q_layer, q_sequence; /* strides in elements, multiples of 8 (of a dimension of one: any) */
    const void *k;             /* bf16 [layers, sequences, positions, kv_heads * dim], 16-byte aligned */
    int64_t k_layer, k_sequence;
    float *weights;            /* [layers, sequences, kv_heads, positions] */
    int64_t w_layer, w_sequence, w_head;
    void *workspace;           /* mkb_key_weights_bytes, 256-byte aligned */
    size_t workspace_bytes;
    int32_t *status;           /* 16 words that a wait which gives up (not all has been added then) writes to (code, ...), or NULL: not recorded */
    uint32_t wait_timeout_ms;  /* of a wait for a launch's own copies and products; 0: 2000 */
    uint32_t reserved;
} MkbsKeyWeights;
size_t mkb_key_weights_bytes(const MkbsKeyWeights *w); /* 0: not valid */
int mkb_key_weights(const MkbsKeyWeights *w, void *cuda_stream);

/*
 * Rows that stay when a sequence of n rows is cut to `keep`: all of them if n <= keep, else its first `sinks`, its last
 * `recent`, and of the others those of the largest weight (equal weights: the lowest row; not a number counts as minus
 * infinity).  rows[..., 0 .. min(n, keep) - 1] are they, ascending; -1 behind them.
 */
typedef struct MkbsSelect {
    uint32_t struct_bytes;
    int32_t layers, sequences, kv_heads;
    int32_t positions;         /* weights per head */
    int32_t length;            /* as in MkbsKeyWeights */
    int32_t keep, sinks, recent; /* sinks + recent <= keep */
    int32_t reserved;
    const int32_t *lengths;
    const float *weights;
    int64_t w_layer, w_sequence, w_head; /* strides in elements */
    int32_t *rows;             /* [layers, sequences, kv_heads, keep] */
    float *kept;               /* NULL, or the weights of these rows in the same order, strides as `weights`; may be `weights` itself */
} MkbsSelect;
int mkb_select_rows(const MkbsSelect *s, void *cuda_stream);

/*
 * Cache row r of every key/value head <- its row rows[r], r = 0 .. min(n, keep) - 1, in place.  `rows` as mkb_select_rows gives
 * them: ascending.  An entry outside the sequence's rows or below r leaves row r as it is.
 */
typedef struct MkbsMove {
    uint32_t struct_bytes;
    int32_t layers, sequences, kv_heads;
    int32_t positions, length, keep;
    int32_t head_bytes;        /* one head's part of a row: a multiple of 16, at most 1024 */
    const int32_t *lengths;    /* rows before the move */
    const int32_t *rows;
    void *caches[2];           /* [layers, sequences, positions, kv_heads, head], 16-byte aligned; the second may be NULL */
    int64_t c_layer, c_sequence; /* strides in bytes, multiples of 16 (of a dimension of one: any) */
} MkbsMove;
int mkb_move_rows(const MkbsMove *m, void *cuda_stream);

/* Message of the last error raised on the calling thread. */
const char *mkb_sequences_last_error(void);
int mkb_sequences_abi_version(void);
/* sizeof of the structs above: 0 beams, 1 region, 2 reorder, 3 key weights, 4 select, 5 move */
size_t mkb_sequences_struct_bytes(int32_t which);

#ifdef __cplusplus
}
#endif
#endif /* MKB200_SEQUENCES_H */
