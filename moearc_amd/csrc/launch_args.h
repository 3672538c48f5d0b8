// Kernel-argument blocks shared by the host runtime (runtime.cpp) and the device code. Plain
// C++ with fixed-width types only, so the host side compiles without the HIP device headers.
#pragma once

#include <stdint.h>

#define MOEARC_KV_F32 0u
#define MOEARC_KV_F16 1u

// Largest number of sequences one decode launch carries in its kernel arguments; the host splits
// larger batches into several launches.
#define MOEARC_MAX_SEQS_PER_LAUNCH 64


// Partial results of a split decode, written by the split kernel when a sequence's span is split
// across work items (one work item = one split of one sequence) and combined by the merge kernel.
// Head-major, so the records of one query head are contiguous:
//   rec_o[(h * n_items + item) * D + d]    un-normalised output (f32), D = 64 or 128 channels
//   rec_ml[(h * n_items + item) * 2 + 0/1] running max (log2 domain) / denominator (f32)
#define MOEARC_MERGE_THREADS 256

// Floats of the code object's fixed record array (moearc_decode_scratch, 8 MiB), which the
// allocation-free decode entry point uses in place of the context's workspace: n_heads * work items
// * (head_dim + 2) floats must fit (64 heads of 64: up to 496 work items; the planner's default is at
// most 128).
#define MOEARC_DECODE_SCRATCH_FLOATS (1u << 21)

// Set in the split kernel's geometry word geo0 (above the page shift, at most 30) when every sequence
// of the launch has as many work items as sequence 0.
#define MOEARC_DECODE_UNIFORM 0x8000u
// Set there when the launch has more than 24 sequences.
#define MOEARC_DECODE_MANY 0x4000u

// Kernel arguments of the split-K decode that are not preloaded scalars (the leading kernel
// arguments carry the KV and block-table bases, q, sequence 0's span, split and item count, and
// the geometry). Passed by value; the per-sequence arrays let one launch serve a ragged batch.
// Work item `it` (one (sequence, split) pair) covers the work-groups it * nkb + kbi for every
// KV-head block kbi, so consecutive work-groups -- which the dispatcher places on consecutive XCDs
// -- take consecutive KV-head blocks of the same split.
struct DecodeArgs {
    const float *q;               // [n_seqs][n_heads][D] f32
    const uint32_t *block_tables; // row b at block_tables + b * bt_stride
    const float *sinks;           // [n_heads] or null
    void *out;                    // [n_seqs][n_heads][D], f32 or f16
    float *rec_o;                 // partial records (see above)
    float *rec_ml;
    uint64_t bt_stride;
    uint32_t n_items;             // work items of the launch (records per head)
    uint32_t out_f16;
    float scale_log2e;            // scale * log2(e)
    uint32_t n_seqs;
    uint32_t item_begin[MOEARC_MAX_SEQS_PER_LAUNCH + 1]; // first work item of each sequence; entries
                                                         // n_seqs .. the end: the work-item count
    uint32_t kv_begin[MOEARC_MAX_SEQS_PER_LAUNCH];       // key span [kv_begin, n_kv)
    uint32_t n_kv[MOEARC_MAX_SEQS_PER_LAUNCH];
};

// The merge kernel's per-sequence item ranges (sequence 0's end is a preloaded argument). One
// spare entry keeps the kernel's argument block a multiple of 8 bytes, the host struct's size.
struct MergeArgs {
    uint32_t item_begin[MOEARC_MAX_SEQS_PER_LAUNCH + 2];
};

// General decode (any head_dim <= 1024, f32 or f16 KV, any page size, any group).
struct DecodeGeneralArgs {
    const float *q;
    const void *k_pages;
    const void *v_pages;
    const uint32_t *block_tables;
    const float *sinks;
    void *out;
    uint64_t bt_stride;
    uint32_t n_heads;
    uint32_t n_kv_heads;
    uint32_t head_dim;
    uint32_t page_tokens;
    uint32_t kv_type;
    uint32_t out_f16;
    float scale;
    uint32_t n_seqs;
    uint32_t kv_begin[MOEARC_MAX_SEQS_PER_LAUNCH];
    uint32_t n_kv[MOEARC_MAX_SEQS_PER_LAUNCH];
};

// Chunked prefill: query rows ((token, head) pairs of one KV head's group) per work-group and the
// work-group size.
#define MOEARC_PREFILL_ROWS 128        // precise (hi/lo weights) kernels
#define MOEARC_PREFILL_FAST_ROWS 256   // default kernels: 64 rows per wave
#define MOEARC_PREFILL_THREADS 256

// Chunked prefill over f16 paged KV, head_dim 64.
struct PrefillArgs {
    const uint16_t *q;            // [n_q][n_heads][64] f16
    const uint16_t *k_pages;
    const uint16_t *v_pages;
    const uint32_t *block_table;
    const float *sinks;
    void *out;                    // [n_q][n_heads][64] f32 or f16
    uint32_t n_q;
    uint32_t pos0;
    uint32_t n_swa;               // 0 = full causal
    uint32_t n_heads;
    uint32_t n_kv_heads;
    uint32_t group;               // 1, 2, 4 or 8
    uint32_t pt_shift;
    uint32_t out_f16;
    float scale_log2e;
    uint32_t n_qtiles;            // query tiles per KV head
    uint16_t *out_lo;             // with f16 output: also f16(o - hi) here, the low half of the
                                  // chunk product's activation split (default kernels; else null)
    uint32_t pair_half;           // the grid is two work-groups per CU, i and i + pair_half sharing
                                  // one (the dispatcher's order): pair_half; otherwise 0
    float boost_a, boost_b;       // the second work-group of a pair keeps a raised issue priority
                                  // for boost_a * its chunks - boost_b * its partner's chunks
};

// A prefill whose query tiles alone leave compute units idle is split along the keys: tile t (of at
// most MOEARC_PF_MAX_TILES) is cut into item_begin[t + 1] - item_begin[t] pieces of nearly equal
// chunk counts, each a work-group per KV head that leaves the partial results of its 256 rows, and
// moearc_attn_prefill_merge_k combines them:
//   rec_o[((item * n_kv_heads + kvh) * 256 + row) * 64 + d]  un-normalised output (f32)
//   rec_ml[((item * n_kv_heads + kvh) * 256 + row) * 2 + 0/1] reference max / row sum in its frame
// A tile of one piece is finished by its work-group and has no records.
#define MOEARC_PF_MAX_TILES 64
#define MOEARC_PF_RECORD_FLOATS (MOEARC_PREFILL_FAST_ROWS * 66u)  // one item's records of one KV head
struct PrefillSplitArgs {
    PrefillArgs a;
    float *rec_o, *rec_ml;
    uint32_t n_items;
    uint32_t tile_tokens;         // query tokens per tile
    uint16_t item_begin[MOEARC_PF_MAX_TILES + 4];  // entries n_qtiles .. the end: n_items
};

// RoPE parameters (moearc_rope, moearc_rope_kv_append_chunk): theta_scale = freq_base^(-2/n_dims),
// computed on the host; neox selects the (p, p + n_dims/2) pairing, else (2p, 2p + 1).
// Heads per thread of the RoPE kernels (grid y runs over groups of this many heads).
constexpr uint32_t ROPE_HEADS = 4;

struct RopeParams {
    uint32_t n_dims;
    uint32_t neox;
    float theta_scale;
    float freq_scale;
    float ext_factor;
    float attn_factor;
    float corr_lo;
    float corr_hi;
};

// ---- quantised matrix-vector products (matvec.hip) ----------------------------------------------
//
// The weight formats, by GGUF type id: bytes per block (BB), elements per block (BE) and elements
// per "piece" (PE) -- the share of a row one lane decodes at a time. A lane owns the pieces
// lane, lane + 64, ... of every row, so the activation values of its pieces stay in registers
// while it walks the rows; MOEARC_MV_PPL_MAX bounds its pieces per pass (a row with more is
// walked in several column slabs).
#define MOEARC_MV_MAX_SEG 32   // matrices (or projections) one launch carries
#define MOEARC_MV_MAX_WAVES 8

constexpr uint32_t moearc_mv_bb(uint32_t ty) {
    return ty == 0 ? 4u : ty == 1 ? 2u : ty == 8 ? 34u : ty == 12 ? 144u : ty == 13 ? 176u
         : ty == 14 ? 210u : ty == 39 ? 17u : 0u;
}
constexpr uint32_t moearc_mv_be(uint32_t ty) {
    return ty == 0 || ty == 1 ? 1u : ty == 8 || ty == 39 ? 32u : ty == 12 || ty == 13 || ty == 14 ? 256u : 0u;
}
constexpr uint32_t moearc_mv_pe(uint32_t ty) {
    return ty == 0 ? 8u : ty == 12 || ty == 13 || ty == 39 ? 32u : 16u;
}
// Largest pieces per lane per pass: activation registers (PPL * PE) stay at or under 128, so a
// wave keeps at least three waves per SIMD of occupancy.
constexpr uint32_t moearc_mv_ppl_max(uint32_t) {
    return 4u;
}
// 16-byte granules one lane stages per slab (a slab of 64 * PPL pieces, any byte alignment).
constexpr uint32_t moearc_mv_gmax(uint32_t ty, uint32_t ppl) {
    return (uint32_t) ((64ull * ppl * moearc_mv_pe(ty) * moearc_mv_bb(ty) / moearc_mv_be(ty) + 30u + 1023u) / 1024u);
}
// Bytes of one wave's staging buffer for slabs of `slab_bytes`: the granules a slab at any
// alignment spans, plus slack for reads that run past a piece.
constexpr uint32_t moearc_mv_wave_buf(uint64_t slab_bytes) {
    return (uint32_t) (((slab_bytes + 30u + 15u) / 16u) * 16u + 64u);
}

// Segment s covers work-groups [wg_end[s-1], wg_end[s]) and rows [0, rows[s]) of matrix w[s]:
// out[s][r] = sum_c W_s[r][c] * x[s][c] (+ bias[s][r] when bit s of bias_mask is set; bias[s]
// then points at the bias, else at any readable rows[s] floats).
struct MatvecArgs {
    const uint8_t *w[MOEARC_MV_MAX_SEG];
    const float *x[MOEARC_MV_MAX_SEG];
    const float *bias[MOEARC_MV_MAX_SEG];
    float *out[MOEARC_MV_MAX_SEG];
    uint32_t rows[MOEARC_MV_MAX_SEG];
    uint32_t wg_end[MOEARC_MV_MAX_SEG];
    uint64_t row_bytes;
    uint32_t n_seg;
    uint32_t n_cols;
    uint32_t n_pieces;     // pieces per row, ceil(n_cols / PE)
    uint32_t n_slabs;      // column slabs per row
    uint32_t rpw;          // consecutive rows per wave
    uint32_t x_in_lds;     // 1: the activation is staged once per work-group in LDS
    uint32_t x_lds_bytes;  // LDS bytes before the waves' staging buffers
    uint32_t wave_buf;     // LDS bytes of one wave's staging buffer
    uint32_t bias_mask;
    uint32_t res_mask;     // bit s: out[s][r] += the result (the residual add), else out[s][r] = it
};

// Chunk-form projections (matmul.hip, matmul2.hip): Y[t][r] = sum_c W[r][c] X[t][c] (+ bias[r]) for
// the n_tok tokens of a prompt chunk, W Q8_0 (8), F16 (1), Q4_K (12), Q5_K (13), Q6_K (14) or
// MXFP4 (39), X given as its f16 hi + lo split. One launch serves up to MOEARC_MM_MAX_SEG matrices
// of one weight type over the same X (a block's q, k and v): its row tiles (grid x) run over the
// segments in order.
#define MOEARC_MM_TOKENS 64    // tokens per work-group
#define MOEARC_MM_MAX_SEG 3
#define MOEARC_MM_SMALL_WAVES 8 // waves per work-group of matmul_small.hip
struct MatmulSeg {
    const uint8_t *w;
    const float *bias;         // [rows] or null
    float *y;                  // [n_tok][y_stride]
    uint64_t row_bytes;
    uint64_t part_off;         // split launches: this matrix's sums at part + z * part_stride + part_off
    uint32_t rows, y_stride;
    uint32_t tile_end;         // row tiles of the launch up to and including this matrix's
    uint32_t pad;
};
struct MatmulArgs {
    MatmulSeg seg[MOEARC_MM_MAX_SEG];
    const uint16_t *xh, *xl;   // [n_tok][cols] f16: x = hi + lo to within 2^-22 |x| or 2^-25
    const float *xs;           // Q4_K, Q5_K: block sums of x, f32 [n_tok][cols / 32] (matmul.hip) or f16
                               // pieces [n_tok][cols / 256][4][8] (matmul2k.hip); matmul_small.hip: x
                               // itself, f32 [n_tok][cols]; else unread
    float *part;               // split launches (grid z > 1): slice z's sums, [t][r] per matrix
    uint64_t part_stride;      // floats per slice: the sum of n_tok * rows over the matrices
    uint32_t n_seg, cols, n_tok;
    uint32_t accumulate;       // 1: y[t][r] += the result (the residual add), else y[t][r] = it
    uint32_t kb_per;           // k-blocks (of 32) per k-slice: work-group z takes blocks kb_per * z ..
                               // (matmul_small.hip: wave w, kb_per * w ..)
    uint32_t pad;
};

// ---- norms with the residual update (norm.hip) --------------------------------------------------
// A row of up to 16 * threads columns stays in its threads' registers (16, 64, 256 or 1024 threads).
#define MOEARC_NORM_PER_THREAD 16u
struct NormArgs {
    void *x;               // [n_rows][n_cols] f32 or f16, or null
    float *h;              // [n_rows][n_cols], updated when y is given
    const void *y;         // [n_rows][n_cols] f32 or f16, or null
    const float *w_post;   // [n_cols] or null: y enters as it is
    const float *gate;     // row r at gate + r * gate_stride, or null
    const float *w_pre;    // [n_cols] or null
    uint64_t gate_stride;
    uint32_t n_rows, n_cols;
    float scale, eps;
    uint32_t x_f16, y_f16;
};

// ---- the router and the experts' products (moe.hip, moe_small.hip, moe_tile.hip) ------------------
#define MOEARC_NO_EXPERT 0xFFFFFFFFu  // a slot without an expert (moearc_attn.h)
#define MOEARC_MAX_EXPERTS 1024u
#define MOEARC_ROUTE_LANES 16u        // lanes per token

struct RouteArgs {
    const float *logits;   // [n_tok][n_expert]
    uint32_t *ids;         // [n_tok][n_used]
    float *weights;        // [n_tok][n_used]
    uint32_t n_tok, n_expert, n_used, over_all;
    float scale;
    uint32_t pad;
};

// A slot is a token's j-th expert, slot t * n_used + j. The plan groups the slots of a call by expert
// in tiles of at most `tile` slots: tiles[i] = (expert, first place, slots; which of its expert's tiles, and
// of how many), list[place] = slot, each expert's slots in their order. Slots without a valid expert form a
// last group, "expert" n_expert.
struct MoeTile {
    uint32_t expert, first;
    uint16_t count, pad;
    uint16_t index, of;
};
// x as moe_tile.hip's products take it: f16 hi (and lo, of f32), each k-block in the order of weights of `type`
struct MoePrepArgs {
    const void *x;
    uint16_t *hi, *lo;
    uint64_t n;                // elements, a multiple of 32
    uint32_t type, pad;
};
struct MoePlanArgs {
    const uint32_t *ids;   // [n_slots]
    MoeTile *tiles;
    uint32_t *n_tiles;
    uint32_t *list;        // [n_slots]
    uint32_t *err;         // set to 1 when an id is neither an expert nor MOEARC_NO_EXPERT
    uint32_t n_slots, n_expert, tile, pad;
    MoePrepArgs prep;          // for the kernels that do both
};

// One grouped product: rows of the experts' matrices times their slots' inputs. With two matrices (gate
// and up) the output is their activation, else the product itself.
struct MoeArgs {
    const uint32_t *ids;       // [n_slots], for launches without a plan (n_slots <= 64)
    const MoeTile *tiles;      // the plan, or null
    const uint32_t *n_tiles, *list;
    const void *x, *x_lo;      // row of slot s: s / x_div; f32 or f16 (x_lo: the f16 halves' low half)
    const uint8_t *w[2];       // expert e's matrix at w + e * expert_bytes
    const float *bias[2];      // [n_expert][rows] or null
    void *y, *y_lo;            // [n_slots][rows]
    uint32_t *err;
    uint64_t expert_bytes, row_bytes;
    uint32_t n_slots, n_expert, x_div, rows, cols;
    uint32_t kb_per;           // moe_small.hip: k-blocks per wave
    uint32_t y_f16;
    uint32_t zero_skipped;     // write zero rows for slots without an expert
    uint32_t clamped;          // the activation: 0 silu(g) u, 1 min(g, limit) sigmoid(alpha g) (clamp(u) + 1)
    float alpha, limit;
    uint32_t row_tiles;        // moe_tile.hip: row tiles per tile of slots
    uint32_t y_order, pad;     // with two matrices: the type of the next product's weights, which orders y
};

// The two launches of a single token (moe_vec.hip). Wave w of work-group g has rows (g * waves + w) * rpw .. of the
// n_used slots: grid y with gate and up, one after the other in down (rpw * n_used at most 64 there, else 32).
struct MoeVecArgs {
    const uint32_t *ids;       // [n_used], at most 64
    const float *weights;      // [n_used]
    const void *x;             // [cols], or [n_used][cols] f32 or f16
    const uint8_t *w[2];
    const float *bias[2];
    void *y;                   // [n_used][rows], or [rows]
    uint32_t *err;
    uint64_t expert_bytes, row_bytes;
    uint32_t n_used, n_expert, rows, cols;
    uint32_t n_pieces, rpw;
    uint32_t x_lds_bytes, wave_buf;
    uint32_t x_f16, y_f16, accumulate, clamped;
    float alpha, limit;
};

// y[t] (+)= sum_j weights[t][j] part[t * n_used + j] over the slots that have an expert, in order
struct MoeCombineArgs {
    const float *part;         // [n_tok * n_used][cols]
    const float *weights;
    const uint32_t *ids;
    void *y;                   // [n_tok][cols] f32 or f16
    uint32_t n_tok, n_used, n_expert, cols, y_f16, accumulate;
};
// Working memory is bounded by cutting long calls into chunks of tokens of at most this many slots: 32,768 slots of
// 2,880 columns hold 0.4 GB per f32 array, and give each of 128 experts 256 slots.
#define MOEARC_MOE_CHUNK_SLOTS 32768u
#define MOEARC_MOE_SMALL_SLOTS 64u  // most slots of a launch without a plan
#define MOEARC_MOE_SMALL_WAVES 8
#define MOEARC_MOE_SMALL_TOKENS 16u
#define MOEARC_MOE_TILE 64u         // most slots of a plan's tile, and of a light one
#define MOEARC_MOE_LIGHT 32u

// ---- ragged batches (append.hip, attn_batch.hip) -------------------------------------------------
//
// Sequences one launch carries in its kernel arguments; the host splits larger batches.
#define MOEARC_BATCH_SEQS 64

// New tokens' q, k and v rows: norm, rotation, q out, K and V into their pages. Row t of the launch (t counts
// from its first sequence's first row) belongs to sequence b, the last one with row_begin[b] <= t.
struct QkvAppendArgs {
    const void *q, *k, *v;          // of the launch's first row, f32 or f16
    const float *q_norm, *k_norm;   // [head_dim] or null
    const float *factors;           // [n_rot / 2] or null
    void *q_out, *k_pages, *v_pages;
    const uint32_t *block_tables;   // of the launch's first sequence
    uint32_t *err;
    uint64_t q_stride, k_stride, v_stride, bt_stride;
    double log2_step;               // -2 log2(freq_base) / n_rot: pair p turns at 2^(p log2_step) radians a position
    float freq_scale, ext_factor, mscale, corr_lo, corr_hi, eps;
    uint32_t n_heads, n_kv_heads, head_dim, n_rot, neox;
    uint32_t in_f16, q_f16, kv_f16, n_pages, page_tokens;
    uint32_t row_off;               // the first work-group's row
    uint32_t pad;
    uint32_t row_begin[MOEARC_BATCH_SEQS];  // entries n_seqs .. the end: 2^32 - 1
    uint32_t n_new[MOEARC_BATCH_SEQS];
    uint32_t n_kv[MOEARC_BATCH_SEQS];
};

// Attention of a ragged batch. A sequence's rows (token, head of the KV head's group) are cut into tiles of 128 or 32
// rows, a tile's keys into pieces; a work-group takes one piece of one tile for one KV head. A slot's work items (tiles x
// pieces) start at item_begin; a slot with more than one piece to a tile leaves records that the merge kernel joins (tr:
// rows of a tile):
//   rec_o[(rec_begin + (tile * pieces + piece) * tr) * n_kv_heads + kvh * tr + row][head_dim]  un-normalised (f32)
//   rec_ml[the same row index][2]   reference max (log2 domain), row sum in its frame
#define MOEARC_AB_ROWS 128u       // rows of a tile: 32 to a wave
#define MOEARC_AB_PT 2016u        // keys' places that a work-group holds at a time (of eight keys each where pages allow): whole
                                  // tiles of 32, or a segment's last tile would hold keys that the next one adds again
#define MOEARC_AB_LOG2_PSCALE 7.0f  // weights are 2^7 at the reference max: f16 keeps 21 bits below it
struct AttnBatchSlot {
    uint32_t item_begin, n_tiles, n_new, n_kv;
    uint32_t seq, row0;             // block-table row; first token's row of q and out
    uint32_t pieces, piece;         // of a tile's keys; keys each, a multiple of 32
    uint32_t rec_begin, merge_begin;  // rows of records, per KV head; tiles that need a merge
    uint32_t tile_rows, pad;
};
struct AttnBatchArgs {
    const uint16_t *q, *k_pages, *v_pages;
    const uint32_t *block_tables;
    const float *sinks;
    uint64_t bt_stride;
    uint32_t n_slots, n_kv_heads, kv_magic, kv_shift;  // x / n_kv_heads = x * magic >> shift for x < 2^31; so
    uint32_t group, group_magic, group_shift;          // the group
    uint32_t page_tokens, page_magic, page_shift;      // and page_tokens
    uint32_t n_swa, n_heads, head_dim;
    uint32_t eights;                // pages of a multiple of eight tokens
    uint32_t n_pages;
    float scale_log2e;
    void *out;
    float *rec_o, *rec_ml;
    uint32_t *err;
    uint32_t out_f16, pad;
    uint32_t item_begin[MOEARC_BATCH_SEQS];   // entries n_slots .. the end: the item count
    uint32_t merge_begin[MOEARC_BATCH_SEQS];
    AttnBatchSlot slot[MOEARC_BATCH_SEQS];
};
