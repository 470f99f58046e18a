// Argument blocks of the kernels for several sequences over paged caches (batch.hip), shared
// with the host runtime.
#ifndef SLM_BATCH_H
#define SLM_BATCH_H

#include <stdint.h>

#define SLM_PG_KEYS 256     // keys of a superblock: one workgroup's, whatever the batch
#define SLM_MOVES_HERE 256  // moves of a sequence and key head that need no launch of their own
#define SLM_MOVES_WG 64     // moves of a workgroup of such a launch
#define SLM_TOP_MAX 32      // alternatives of a row of logits
#define SLM_FEW_IDS 256     // tokens that go to the kernel with its arguments
#define SLM_NO_SEQ 0xffffffffu

// A batch of sequences on the device (slm_seqs).
struct SeqsDev {
    const uint32_t* len;     // [n] tokens in the pages
    const uint32_t* seen;    // [n] tokens ever: the newest one's position + 1
    const uint32_t* first;   // [n + 1] rows of new tokens before each sequence's
    const uint32_t* ifirst;  // [n + 1] superblocks before each sequence's (one at least each)
    const uint32_t* items;   // [items][4] sequence (SLM_NO_SEQ: none), superblock of it, its length, 0
    const uint32_t* table;   // [n][width] pages
    int32_t n, width;
};

struct PStoreArgs {
    SeqsDev s;
    void *k, *v;             // [pages][kh][page][dh], fp32 or fp16
    float* mass;             // [pages][kh][page] or null
    uint32_t* born;          // likewise
    const float *ksrc, *vsrc;  // [rows][kh][dh]
    int32_t rows, kh, page, dh;
    int32_t each;            // one new token in every sequence: row b is sequence b's
};

struct PAttnArgs {
    SeqsDev s;
    float* y;                // [n][heads][dh]
    const float* q;
    const void *k, *v;
    const float* mass;       // with mass_out
    float* mass_out;         // or null
    const uint32_t* born;    // positions, or null: slot t holds position t
    float* ml;               // [heads][items][2] maximum (powers of two) and sum
    float* po;               // [items][heads][dh] weighted values
    float* sc;               // [items][heads][SLM_PG_KEYS] scores, with mass_out
    int32_t items;
    int32_t heads, kh, page, dh;
    int64_t gap;
    float scale;             // times log2 e
    int32_t direct;          // every sequence is one superblock: no join
    int32_t r16;             // fp16 mode: y rounded to fp16
};

struct PEvictArgs {
    SeqsDev s;
    void *k, *v;
    const float* mass;
    const uint32_t* born;
    float* mass_out;
    uint32_t* born_out;
    uint32_t* moves;         // [n·kh][2][most] slots left, slots that move there
    uint32_t* count;         // [n·kh] moves; null: at most SLM_MOVES_HERE, made by the launch that finds them
    int32_t kh, page, dh;
    uint32_t keep, recent, most;
    int32_t in_place;        // mass_out is mass and born_out is born
    int32_t unit;            // bytes of a value
    uint32_t room;           // slots whose keys LDS has room for, a multiple of 64
    int32_t vec;             // mass and born can be read four slots at a time
};

struct PMoveArgs {
    PEvictArgs e;
    uint32_t blocks;         // workgroups a (sequence, key head)
};

struct LogpArgs {
    const float* x;          // [m][n]
    const uint32_t* ids;     // [m], or null: in `few`
    float *lp, *ent;         // [m]; ent may be null
    uint32_t* top_ids;       // [m][top]
    float* top_lp;
    int64_t m, n;
    int32_t top;
    int32_t parts, span;     // workgroups of a row, and the logits of each
    float* part_sums;        // [m][parts][4]
    uint64_t* part_top;      // [m][parts][top], best first
    uint32_t few[SLM_FEW_IDS];  // up to this many rows' tokens, outside a recorded step
};

#endif
