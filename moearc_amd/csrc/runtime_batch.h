// The host side of the ragged batches' calls (append.hip, attn_batch.hip): included at the end of runtime.cpp, whose
// launch, workspace and profiling helpers it uses.
#pragma once

namespace {

constexpr unsigned long kBatchRows = 1ul << 20;  // new tokens of a call: launches stay below 2^32 threads
constexpr unsigned long kBatchHeads = 1024;

bool batch_load(moearc_ctx *c) {
    struct {
        hipFunction_t *slot;
        const char *name;
    } fns[] = {
        {&c->f_qkv_append[0][0], "moearc_qkv_append_l8_k"},  {&c->f_qkv_append[0][1], "moearc_qkv_append_l8x3_k"},
        {&c->f_qkv_append[1][0], "moearc_qkv_append_l16_k"}, {&c->f_qkv_append[1][1], "moearc_qkv_append_l16x3_k"},
        {&c->f_qkv_append[2][0], "moearc_qkv_append_l32_k"}, {&c->f_qkv_append[2][1], "moearc_qkv_append_l32x3_k"},
        {&c->f_qkv_append_any, "moearc_qkv_append_any_k"},
        {&c->f_attn_batch[0][0], "moearc_attn_batch_d2_k"}, {&c->f_attn_batch[0][1], "moearc_attn_batch_precise_d2_k"},
        {&c->f_attn_batch[1][0], "moearc_attn_batch_d4_k"}, {&c->f_attn_batch[1][1], "moearc_attn_batch_precise_d4_k"},
        {&c->f_attn_batch[2][0], "moearc_attn_batch_d8_k"}, {&c->f_attn_batch[2][1], "moearc_attn_batch_precise_d8_k"},
        {&c->f_attn_batch_merge, "moearc_attn_batch_merge_k"},
    };
    for (auto &f : fns)
        if (hipModuleGetFunction(f.slot, c->module, f.name) != hipSuccess) {
            std::fprintf(stderr, "moearc: code object lacks kernel %s\n", f.name);
            return false;
        }
    return true;
}

// The sequences of a call: new tokens row_begin[b] .. row_begin[b + 1] - 1, the last of n_kv[b] keys, which the block
// table's row holds.
int batch_check(const unsigned int *row_begin, const unsigned int *n_kv, unsigned long n_seqs, unsigned long bt_stride,
                unsigned long page_tokens) {
    for (unsigned long b = 0; b < n_seqs; ++b) {
        if (row_begin[b + 1] < row_begin[b] || n_kv[b] >= (1u << 30)) return ERR_ARG;
        if (row_begin[b + 1] != row_begin[b] && (n_kv[b] + page_tokens - 1) / page_tokens > bt_stride) return ERR_ARG;
    }
    return n_seqs && row_begin[n_seqs] > kBatchRows ? ERR_ARG : OK;
}

// A call that may set the error word: the next moearc_sync reads it, every one once a graph holds such a call.
void batch_arm(moearc_ctx *c) {
    if (capturing(c)) c->err_in_graph = true;
    else c->err_armed = true;
}

// ---- attention ------------------------------------------------------------------------------------

// What the plan of a group of sequences (at most MOEARC_BATCH_SEQS) needs to know of the call.
struct BatchShape {
    unsigned long n_swa, group, n_kv_heads, head_dim;
    unsigned cus, wgs;  // work-groups that the device holds at once
};

struct BatchSeq {
    uint32_t seq, row0, n_new, n_kv;
};

struct BatchPlan {
    uint32_t n = 0, items = 0, merge_tiles = 0, merge_rows = 0;
    uint64_t records = 0;  // rows of records, per KV head
    BatchSeq s[MOEARC_BATCH_SEQS];
    uint32_t tile_rows[MOEARC_BATCH_SEQS], n_tiles[MOEARC_BATCH_SEQS], pieces[MOEARC_BATCH_SEQS], piece[MOEARC_BATCH_SEQS];
};

// The 32-key chunks of a sequence's tiles (attn_batch.hip's ab_span): at most `longest` in one, about `sum` in all.
struct BatchWork {
    uint64_t longest, sum;
};
BatchWork batch_work(const BatchSeq &s, const BatchShape &sh, uint64_t tile_rows, uint64_t n_tiles) {
    const int64_t shift = (int64_t) s.n_kv - s.n_new;
    auto chunks = [&](uint64_t last_row) {  // without a window, up to this row's token
        const int64_t hi = shift + std::min<int64_t>((int64_t) (last_row / sh.group), (int64_t) s.n_new - 1) + 1;
        return hi > 0 ? (uint64_t) (hi + 31) / 32 : 0ull;
    };
    const uint64_t first = chunks(tile_rows - 1), last = chunks(n_tiles * tile_rows - 1);
    // a window's keys, those of a tile's other tokens, and up to seven that the first page of eights has before them
    const uint64_t window = sh.n_swa ? (sh.n_swa + (tile_rows + sh.group - 1) / sh.group + 7 + 31) / 32 : ~0ull;
    return BatchWork{std::max<uint64_t>(1, std::min(last, window)), n_tiles * std::min((first + last + 1) / 2, window)};
}

// Sequences from `at` on that one launch carries; those without new tokens are passed over. The ones with the most keys
// come first, so that their work-groups start first.
unsigned long batch_take(BatchPlan &p, const unsigned int *row_begin, const unsigned int *n_kv, unsigned long n_seqs, unsigned long at) {
    p.n = 0;
    for (; at < n_seqs && p.n < MOEARC_BATCH_SEQS; ++at)
        if (row_begin[at + 1] != row_begin[at])
            p.s[p.n++] = BatchSeq{(uint32_t) at, row_begin[at], row_begin[at + 1] - row_begin[at], n_kv[at]};
    std::sort(p.s, p.s + p.n, [](const BatchSeq &x, const BatchSeq &y) { return x.n_kv != y.n_kv ? x.n_kv > y.n_kv : x.seq < y.seq; });
    return at;
}

// Tiles: of 128 rows, their waves in step on the same keys, or of 32, each wave with keys of its own, which read K and V
// once per tile as well. The latter for a sequence of up to 64 rows, and where full tiles would leave half of the CUs
// without work, for one of up to 256 rows or 2560 keys. Measured, full and small tiles, us: 64 heads over 8 KV heads of 64 channels,
// four sequences of 16 tokens behind 1500 20.2 and 16.8, of 32 tokens 21.0 and 19.5; 32 such sequences 45.4 and 47.4, 49.6 and 77.3; 64
// behind 100, 13.9 and 23.5; one of 200 behind 800 23.1 and 16.7. 32 heads over 4 of 128, one of 300 15.8 and 13.2, of 500 behind
// 2000 44.6 and 40.5, of 100 behind 16,000 48.9 and 53.2, of 512 behind 32,700 304 and 390, two of 128 behind 4000 37.8 and 41.2.
// The limit of 2560 keys, 32 heads over 4 of 128, one sequence of 200, 300 and 500 tokens: behind 1000 27.6 and 24.7, 28.6 and 23.6, 38.2 and 26.5; behind
// 3000 33.5 and 34.7, 37.4 and 40.8, 50.3 and 49.5; behind 6000 45.8 and 47.4, 52.4 and 68.2, 75.0 and 82.1. Other heads put the
// border elsewhere, 8 over 1 of 128 at 6000 and 16 over 2 of 256 at 2000 for 300 tokens. 33 to 64 rows, one half-empty full tile or
// two small ones: 64 heads over 8 of 64, 5 to 8 tokens behind 2000, 8 sequences 18 and 18 to 22, 32 40 and 32, 64 66 and 73;
// 32 behind 8000 124 and 137; 32 over 4 of 128, up to 32 sequences the same to 4%, 64 behind 2000 74 and 85.
// Pieces: where a tile's keys would keep one work-group longer than the whole work keeps the device; with fewer, all
// work-groups run at once and the longest decides. Work is counted in 32-key chunks of a small tile, whose work-group takes four
// at a time; a full tile's takes one. A piece has at least four of these steps, a full tile's sixteen: drafts of 3 to 7 tokens behind
// 500 to 3000 take 15.5 us, 15.2 with half as many, 20.3 with twice; a full tile's pieces of eight chunks cost 2 us of 30.
void batch_plan(BatchPlan &p, const BatchShape &sh, bool may_split) {
    uint64_t total = 0, most = 0, longest[MOEARC_BATCH_SEQS], full_wgs = 0;
    for (uint32_t i = 0; i < p.n; ++i)
        full_wgs += ((uint64_t) p.s[i].n_new * sh.group + MOEARC_AB_ROWS - 1) / MOEARC_AB_ROWS * sh.n_kv_heads;
    const bool idle = 2 * full_wgs <= sh.cus;
    for (uint32_t i = 0; i < p.n; ++i) {
        const uint64_t rows = (uint64_t) p.s[i].n_new * sh.group;
        p.tile_rows[i] = rows <= 64 || (idle && (rows <= 256 || p.s[i].n_kv <= 2560)) ? 32u : MOEARC_AB_ROWS;
        p.n_tiles[i] = (uint32_t) ((rows + p.tile_rows[i] - 1) / p.tile_rows[i]);
        const BatchWork w = batch_work(p.s[i], sh, p.tile_rows[i], p.n_tiles[i]);
        longest[i] = w.longest;
        const uint64_t cost = p.tile_rows[i] == MOEARC_AB_ROWS ? 4 : 1;
        total += w.sum * cost;
        most = std::max(most, longest[i] * cost);
    }
    uint64_t even = std::max<uint64_t>(16, (total * sh.n_kv_heads + sh.wgs - 1) / sh.wgs);
    const bool split = may_split && most > even + even / 4;
    // Pieces that together are a few more than the device holds at once would run in a second round: longer ones.
    auto cut = [&](uint32_t i) {
        const bool full = p.tile_rows[i] == MOEARC_AB_ROWS;
        const uint64_t chunks = full ? std::max<uint64_t>((even + 3) / 4, 16) : (even + 3) / 4 * 4;
        const bool whole = !split || longest[i] <= chunks + chunks / 4;
        p.piece[i] = whole ? 0x40000000u : (uint32_t) std::min<uint64_t>(chunks * 32, 0x40000000u);
        p.pieces[i] = whole ? 1u : (uint32_t) ((longest[i] * 32 + p.piece[i] - 1) / p.piece[i]);
        return (uint64_t) p.n_tiles[i] * p.pieces[i];
    };
    for (int k = 0; k < 8; ++k) {
        uint64_t wgs = 0;
        for (uint32_t i = 0; i < p.n; ++i) wgs += cut(i) * sh.n_kv_heads;
        if (!split || wgs <= sh.wgs || wgs >= 2 * sh.wgs) break;
        even += even / 16 + 1;
    }
    p.items = p.merge_tiles = p.merge_rows = 0;
    p.records = 0;
    for (uint32_t i = 0; i < p.n; ++i) {
        p.items += p.n_tiles[i] * p.pieces[i];
        if (p.pieces[i] > 1) {
            p.records += (uint64_t) p.n_tiles[i] * p.pieces[i] * p.tile_rows[i];
            p.merge_tiles += p.n_tiles[i];
            p.merge_rows = std::max(p.merge_rows, p.tile_rows[i]);
        }
    }
}

size_t batch_record_bytes(const BatchPlan &p, const BatchShape &sh) {
    return (size_t) p.records * sh.n_kv_heads * (sh.head_dim + 2) * sizeof(float);
}

// x / d for x below 2^31 as x * magic >> shift: with 2^s >= d, ceil(2^(31 + s) / d) is off by less than 2^-s
// relative, so the quotient is exact.
void batch_divisor(unsigned long d, uint32_t &magic, uint32_t &shift) {
    const uint32_t s = log2u(d);
    magic = (uint32_t) (((1ull << (31 + s)) + d - 1) / d);
    shift = 31 + s;
}

// The checks that the attention and its workspace share.
int attn_batch_check(unsigned long n_heads, unsigned long n_kv_heads, unsigned long head_dim, unsigned long n_swa) {
    if (n_heads == 0 || n_heads > kBatchHeads || n_kv_heads == 0 || n_heads % n_kv_heads != 0) return ERR_ARG;
    if (head_dim == 0 || head_dim % 8 != 0 || head_dim > 256 || n_swa >= (1ul << 31)) return ERR_ARG;
    return OK;
}

BatchShape batch_shape(const moearc_ctx *c, unsigned long n_heads, unsigned long n_kv_heads, unsigned long head_dim, unsigned long n_swa) {
    const unsigned cu = c->n_cu ? c->n_cu : 256;
    return BatchShape{n_swa, n_heads / n_kv_heads, n_kv_heads, head_dim, cu, cu * (head_dim <= 64 ? 3u : head_dim <= 128 ? 2u : 1u)};
}

}  // namespace

extern "C" {

int moearc_rope_qkv_append_batched(moearc_ctx *c, const moearc_qkv_append *d, const unsigned int *block_tables,
                                   unsigned long bt_stride, const unsigned int *row_begin, const unsigned int *n_kv,
                                   unsigned long n_seqs) {
    if (!c || !d || !block_tables || !row_begin || !n_kv) return ERR;
    if (!d->q || !d->k || !d->v || !d->q_out || !d->k_pages || !d->v_pages) return ERR;
    if (d->in_type > 1 || d->q_type > 1 || d->kv_type > 1) return ERR_ARG;
    if (d->n_heads == 0 || d->n_heads > kBatchHeads || d->n_kv_heads == 0 || d->n_kv_heads > kBatchHeads) return ERR_ARG;
    const unsigned long D = d->head_dim;
    if (D == 0 || D > 2 * 128 || d->n_rot == 0 || d->n_rot % 2 != 0 || d->n_rot > D) return ERR_ARG;
    if (d->page_tokens == 0 || d->page_tokens > (1ul << 30) || d->n_pages == 0 || d->n_pages > (1ul << 32) - 1) return ERR_ARG;
    if (d->q_stride < d->n_heads * D || d->k_stride < d->n_kv_heads * D || d->v_stride < d->n_kv_heads * D) return ERR_ARG;
    if (d->q_stride >= (1ul << 40) || d->k_stride >= (1ul << 40) || d->v_stride >= (1ul << 40)) return ERR_ARG;
    if (!(d->freq_base > 0.f && d->freq_base <= 3.0e38f) || !(d->freq_scale > 0.f) || !((d->q_norm || d->k_norm) ? d->eps >= 0.f : true))
        return ERR_ARG;
    if (const int rc = batch_check(row_begin, n_kv, n_seqs, bt_stride, d->page_tokens)) return rc;
    if (n_seqs == 0 || row_begin[n_seqs] == row_begin[0]) return OK;
    QkvAppendArgs a{};
    a.q_norm = d->q_norm;
    a.k_norm = d->k_norm;
    a.factors = d->freq_factors;
    a.k_pages = d->k_pages;
    a.v_pages = d->v_pages;
    a.err = c->err_word;
    a.q_stride = d->q_stride;
    a.k_stride = d->k_stride;
    a.v_stride = d->v_stride;
    a.bt_stride = bt_stride;
    a.log2_step = -2.0 * std::log2((double) d->freq_base) / (double) d->n_rot;
    a.freq_scale = d->freq_scale;
    a.ext_factor = d->ext_factor;
    a.mscale = d->attn_factor;
    if (d->ext_factor != 0.f) a.mscale *= 1.0f + 0.1f * std::log(1.0f / d->freq_scale);
    a.corr_lo = d->corr_lo;
    a.corr_hi = d->corr_hi;
    a.eps = d->eps;
    a.n_heads = (uint32_t) d->n_heads;
    a.n_kv_heads = (uint32_t) d->n_kv_heads;
    a.head_dim = (uint32_t) D;
    a.n_rot = (uint32_t) d->n_rot;
    a.neox = d->neox != 0;
    a.in_f16 = d->in_type;
    a.q_f16 = d->q_type;
    a.kv_f16 = d->kv_type;
    a.n_pages = (uint32_t) d->n_pages;
    a.page_tokens = (uint32_t) d->page_tokens;
    const size_t in_size = d->in_type ? 2 : 4, q_size = d->q_type ? 2 : 4, kv_size = d->kv_type ? 2 : 4;
    // Quads: every row of four channels at a multiple of four elements from an aligned base.
    auto quads = [](const void *p, size_t size) { return (uintptr_t) p % (4 * size) == 0; };
    const bool wide = D % 8 == 0 && d->n_rot % 8 == 0 && d->q_stride % 4 == 0 && d->k_stride % 4 == 0 && d->v_stride % 4 == 0 &&
                      quads(d->q, in_size) && quads(d->k, in_size) && quads(d->v, in_size) && quads(d->q_out, q_size) &&
                      quads(d->k_pages, kv_size) && quads(d->v_pages, kv_size) && quads(d->q_norm, 4) && quads(d->k_norm, 4);
    const int kind = D <= 64 ? 0 : D <= 128 ? 1 : 2;
    const uint64_t heads = d->n_heads + 2 * d->n_kv_heads, per_wg = wide ? 32u >> kind : 4u;
    uint64_t groups = (heads + per_wg - 1) / per_wg;
    // A work-group of three heads a thread where those of one would be more than the device holds (eight to a CU).
    const bool many = wide && groups * (row_begin[n_seqs] - row_begin[0]) > 8ull * (c->n_cu ? c->n_cu : 256u);
    if (many) groups = (groups + 2) / 3;
    const hipFunction_t kernel = wide ? c->f_qkv_append[kind][many] : c->f_qkv_append_any;
    const LaunchScope scope(c, "rope_qkv_append", d->n_heads, D);
    batch_arm(c);
    const uint32_t step = (uint32_t) (kMaxThreads / 256 / groups);
    for (unsigned long at = 0; at < n_seqs; at += MOEARC_BATCH_SEQS) {
        const uint32_t cnt = (uint32_t) std::min<unsigned long>(MOEARC_BATCH_SEQS, n_seqs - at), first = row_begin[at];
        const uint32_t rows = row_begin[at + cnt] - first;
        if (rows == 0) continue;
        for (uint32_t i = 0; i < MOEARC_BATCH_SEQS; ++i) {
            a.row_begin[i] = i < cnt ? row_begin[at + i] - first : 0xFFFFFFFFu;
            a.n_new[i] = i < cnt ? row_begin[at + i + 1] - row_begin[at + i] : 0u;
            a.n_kv[i] = i < cnt ? n_kv[at + i] : 0u;
        }
        a.q = (const uint8_t *) d->q + (size_t) first * d->q_stride * in_size;
        a.k = (const uint8_t *) d->k + (size_t) first * d->k_stride * in_size;
        a.v = (const uint8_t *) d->v + (size_t) first * d->v_stride * in_size;
        a.q_out = (uint8_t *) d->q_out + (size_t) first * d->n_heads * D * q_size;
        a.block_tables = block_tables + at * bt_stride;
        for (a.row_off = 0; a.row_off < rows; a.row_off += step)
            if (const int rc = launch2d(c, kernel, std::min(step, rows - a.row_off), (unsigned) groups, 256, a, nullptr,
                                        d->n_heads, D, 0, "rope_qkv_append"))
                return rc;
    }
    return OK;
}

int moearc_attn_prefill_batched_workspace(moearc_ctx *c, const unsigned int *row_begin, const unsigned int *n_kv,
                                          unsigned long n_seqs, unsigned long n_swa, unsigned long n_heads,
                                          unsigned long n_kv_heads, unsigned long head_dim, unsigned long *bytes) {
    if (!c || !row_begin || !n_kv || !bytes) return ERR;
    if (const int rc = attn_batch_check(n_heads, n_kv_heads, head_dim, n_swa)) return rc;
    if (const int rc = batch_check(row_begin, n_kv, n_seqs, ~0ul, 1)) return rc;
    const BatchShape sh = batch_shape(c, n_heads, n_kv_heads, head_dim, n_swa);
    *bytes = 0;
    BatchPlan p;
    for (unsigned long at = 0; at < n_seqs;) {
        at = batch_take(p, row_begin, n_kv, n_seqs, at);
        batch_plan(p, sh, true);
        *bytes = std::max<unsigned long>(*bytes, batch_record_bytes(p, sh));
    }
    return OK;
}

int moearc_attn_prefill_batched(moearc_ctx *c, void *out, unsigned int out_type, const void *q, const void *k_pages,
                                const void *v_pages, unsigned long n_pages, const unsigned int *block_tables,
                                unsigned long bt_stride, const unsigned int *row_begin, const unsigned int *n_kv,
                                const float *sinks, unsigned long n_seqs, unsigned long n_swa, unsigned long n_heads,
                                unsigned long n_kv_heads, unsigned long head_dim, unsigned long page_tokens, float scale,
                                unsigned int kv_type, void *ws, unsigned long ws_bytes) {
    if (!c || !out || !q || !k_pages || !v_pages || !block_tables || !row_begin || !n_kv) return ERR;
    if (kv_type != 1u || out_type > 1u) return ERR_ARG;
    if (const int rc = attn_batch_check(n_heads, n_kv_heads, head_dim, n_swa)) return rc;
    if (page_tokens == 0 || page_tokens > (1ul << 30) || n_pages == 0 || n_pages > (1ul << 32) - 1) return ERR_ARG;
    if (n_pages > 0xFFFFFFFFul / page_tokens) return ERR_ARG;  // places in a pool are 32-bit numbers
    const float c2 = scale * 1.4426950408889634f;
    if (!(std::fabs(c2) <= 3.0e38f)) return ERR_ARG;
    if (((uintptr_t) out | (uintptr_t) q | (uintptr_t) k_pages | (uintptr_t) v_pages) % 16 != 0) return ERR_ARG;
    if (const int rc = batch_check(row_begin, n_kv, n_seqs, bt_stride, page_tokens)) return rc;
    const BatchShape sh = batch_shape(c, n_heads, n_kv_heads, head_dim, n_swa);
    unsigned long need = 0;
    if (const int rc = moearc_attn_prefill_batched_workspace(c, row_begin, n_kv, n_seqs, n_swa, n_heads, n_kv_heads, head_dim, &need))
        return rc;
    if (ws && ((uintptr_t) ws % 16 != 0 || ws_bytes < need)) return ERR_ARG;
    if (n_seqs == 0 || row_begin[n_seqs] == row_begin[0]) return OK;
    bool split = true;
    if (need && !ws) {
        if (capturing(c)) return ERR;
        // without memory for the records every tile is one work-group's
        split = ensure_floats(c, c->ab_ws, c->ab_ws_floats, need / sizeof(float)) == OK;
        ws = c->ab_ws;
    }
    AttnBatchArgs a{};
    a.q = (const uint16_t *) q;
    a.k_pages = (const uint16_t *) k_pages;
    a.v_pages = (const uint16_t *) v_pages;
    a.block_tables = block_tables;
    a.sinks = sinks;
    a.out = out;
    a.err = c->err_word;
    a.bt_stride = bt_stride;
    a.n_swa = (uint32_t) n_swa;
    a.n_heads = (uint32_t) n_heads;
    a.n_kv_heads = (uint32_t) n_kv_heads;
    a.group = (uint32_t) sh.group;
    a.head_dim = (uint32_t) head_dim;
    a.page_tokens = (uint32_t) page_tokens;
    batch_divisor(page_tokens, a.page_magic, a.page_shift);
    batch_divisor(sh.group, a.group_magic, a.group_shift);
    batch_divisor(n_kv_heads, a.kv_magic, a.kv_shift);
    a.eights = page_tokens % 8 == 0;
    a.n_pages = (uint32_t) n_pages;
    a.out_f16 = out_type;
    a.scale_log2e = c2;
    const int kind = head_dim <= 64 ? 0 : head_dim <= 128 ? 1 : 2;
    const LaunchScope scope(c, "attn_prefill_batched", n_heads, row_begin[n_seqs] - row_begin[0]);
    batch_arm(c);
    BatchPlan p;
    for (unsigned long at = 0; at < n_seqs;) {
        at = batch_take(p, row_begin, n_kv, n_seqs, at);
        if (p.n == 0) continue;
        batch_plan(p, sh, split);
        a.n_slots = p.n;
        uint32_t item = 0, merge = 0;
        uint64_t rec = 0;
        for (uint32_t i = 0; i < MOEARC_BATCH_SEQS; ++i) {
            a.item_begin[i] = item;
            a.merge_begin[i] = merge;
            if (i >= p.n) continue;
            a.slot[i] = AttnBatchSlot{item, p.n_tiles[i], p.s[i].n_new, p.s[i].n_kv, p.s[i].seq, p.s[i].row0,
                                      p.pieces[i], p.piece[i], (uint32_t) rec, merge, p.tile_rows[i], 0u};
            item += p.n_tiles[i] * p.pieces[i];
            if (p.pieces[i] > 1) {
                rec += (uint64_t) p.n_tiles[i] * p.pieces[i] * p.tile_rows[i];
                merge += p.n_tiles[i];
            }
        }
        a.rec_o = (float *) ws;
        a.rec_ml = (float *) ws + (size_t) p.records * n_kv_heads * head_dim;
        if (const int rc = launch(c, c->f_attn_batch[kind][out_type == MOEARC_OUT_F32], (unsigned) (p.items * n_kv_heads), 256, a,
                                  nullptr, n_heads, head_dim, "attn_prefill_batched"))
            return rc;
        if (p.merge_tiles) {
            const unsigned at_a_time = 256u / ((unsigned) head_dim / 4u);
            if (const int rc = launch2d(c, c->f_attn_batch_merge, (unsigned) (p.merge_tiles * n_kv_heads),
                                        (p.merge_rows + at_a_time - 1) / at_a_time, 256, a, nullptr, n_heads, head_dim, 0,
                                        "attn_prefill_batched.merge"))
                return rc;
        }
    }
    return OK;
}

}  // extern "C"
