// The host side of the norms and of the experts' half of a block (norm.hip, moe*.hip): included at the
// end of runtime.cpp, whose launch, workspace and profiling helpers it uses.
#pragma once

namespace {

constexpr uint64_t kMaxThreads = 1ull << 31;  // of a launch, which may not have 2^32

constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// The parts of a call's workspace, in order.
struct MoeSpace {
    size_t tiles = 0, list = 0, split = 0, act = 0, part = 0, bytes = 0;
    size_t split_n = 0, act_n = 0;  // elements of x and of the activations
};

uint64_t moe_max_tiles(uint64_t slots, uint64_t n_expert, uint64_t tile) {
    return std::min<uint64_t>(slots, (slots + tile - 1) / tile + n_expert + 1);
}

// Tokens that run at a time: what the plan's LDS holds, and rows no wider than a launch has threads for (up to two a row in
// moe_tile.hip; `widest` counts rows of gate and up twice, of which a tile has half as many).
uint64_t moe_chunk(uint64_t n_used, uint64_t widest) {
    return std::max<uint64_t>(1, std::min<uint64_t>(MOEARC_MOE_CHUNK_SLOTS, kMaxThreads / 2 / std::max<uint64_t>(widest, 1)) / n_used);
}

uint64_t moe_ffn_chunk(uint64_t n_used, uint64_t n_embd, uint64_t n_ff) { return moe_chunk(n_used, std::max(n_embd, 2 * n_ff)); }

// Whether gate and up of one token's slots, a tile each, fit a launch: all sizes but 1024 slots of the widest rows.
bool moe_ffn_fits(uint64_t n_used, uint64_t n_ff) { return n_used * ((n_ff + 63) / 64) * 256 < 2 * kMaxThreads; }

// A call of n_tok tokens (one chunk of it) with n_used experts each: n_ff 0 for a product alone.
MoeSpace moe_space(uint64_t n_tok, uint64_t n_used, uint64_t n_expert, uint64_t n_embd, uint64_t n_ff, uint64_t chunk) {
    const uint64_t tok = std::min<uint64_t>(n_tok, chunk), slots = tok * n_used;
    MoeSpace s;
    s.tiles = 256;
    s.list = s.tiles + align256(sizeof(MoeTile) * moe_max_tiles(slots, n_expert, MOEARC_MOE_LIGHT));
    s.split = s.list + align256(4 * slots);
    s.split_n = (n_ff ? tok : slots) * n_embd;  // a product alone may have a row of x for each slot
    s.act_n = slots * n_ff;
    s.act = s.split + align256(4 * s.split_n);
    s.part = s.act + align256(4 * s.act_n);
    s.bytes = s.part + (n_ff ? align256(4 * slots * n_embd) : 0);
    return s;
}

// The call's working memory: the caller's, or the context's, grown on demand. A captured call takes the
// caller's only: the context's may move with a later call, and is shared by whatever else the context runs.
int moe_take_space(moearc_ctx *c, size_t need, void *ws, uint8_t **out) {
    if (ws) {
        *out = (uint8_t *) ws;
        return OK;  // the size and alignment were checked before anything was enqueued
    }
    if (capturing(c)) return ERR;
    if (const int rc = ensure_floats(c, c->moe_ws, c->moe_ws_floats, (need + 3) / 4)) return rc;
    *out = (uint8_t *) c->moe_ws;
    return OK;
}

// The call's kernels may set the error word, and go on doing so when they were captured.
void moe_arm(moearc_ctx *c, const void *ws) {
    c->err_armed = true;
    if (ws && capturing(c)) c->err_in_graph = true;
}

int moe_space_check(size_t need, const void *ws, unsigned long ws_bytes) {
    return ws && (ws_bytes < need || (uintptr_t) ws % 256 != 0) ? ERR_ARG : OK;
}

constexpr unsigned kMoeTypes[6] = {1, 8, 12, 13, 14, 39};
constexpr const char *kMoeNames[6] = {"f16", "q8_0", "q4_k", "q5_k", "q6_k", "mxfp4"};
int moe_index(unsigned ty) {
    for (int i = 0; i < 6; ++i)
        if (kMoeTypes[i] == ty) return i;
    return -1;
}

bool moe_cols_ok(unsigned long n_cols) { return n_cols >= 256 && n_cols % 32 == 0 && n_cols <= 0x100000ul; }

int moe_matrix_check(unsigned ty, const void *w, unsigned long n_rows, unsigned long n_cols) {
    if (moe_index(ty) < 0 || !moe_cols_ok(n_cols) || n_cols % moearc_mv_be(ty) != 0 || n_rows == 0 || n_rows > 0x100000ul || ((uintptr_t) w & 1u))
        return ERR_ARG;
    return OK;
}

int moe_count_check(unsigned long n_tok, unsigned long n_used, unsigned long n_expert, unsigned int io_type) {
    if (io_type > MOEARC_OUT_F16 || n_expert == 0 || n_expert > MOEARC_MAX_EXPERTS || n_used == 0 ||
        n_used > MOEARC_MAX_EXPERTS || n_tok >= 0x80000000ul)
        return ERR_ARG;
    return OK;
}

// Whether a chunk runs on tiles of 32 slots, not 64: up to 56 slots an expert, 40 with f16 inputs. (Products of 64
// slots an expert, 64 and 32 slots a tile: MXFP4 142 and 121 us, Q8_0 88 and 82, Q4_K 84 and 86, Q5_K 97 and 100, f16
// Q4_K 155 and 166, Q6_K 149 and 157; of 32: MXFP4 87 and 82, Q4_K 69 and 58, Q5_K 80 and 67, f16 Q4_K 111 and 109.)
// One threshold for all types: f32 MXFP4's and Q8_0's lie above it, where was not measured.
bool moe_light(uint64_t n_slots, uint64_t n_expert, bool half) { return n_slots < (half ? 40 : 56) * n_expert; }

// Rows of each matrix that a tile's work-group takes: moe_tile.hip's shapes.
uint32_t moe_tile_rows(unsigned ty, bool half, bool light, bool gate_up) {
    const bool wide = !light && (ty == 12u || ty == 13u || (ty == 39u && !half));
    return (wide ? 256u : 128u) / (gate_up ? 2u : 1u);
}

// Whether a chunk runs without a plan (moe_small.hip): up to 64 slots, which a wave's lanes search, but for more than
// 24 over 32 or more experts of MXFP4. Products of 32 and 64 slots without a plan and on tiles, us: 64 Q4_K experts of
// 2048 x 1024 19, 26 and 23, 24; of Q8_0, 2048 x 2048, 31, 40 and 40, 41; eight 16, 17 and 29, 29; f16 ones of F16 33, 44
// and 34, 44; one of Q5_K, 4096 x 2048, 15, 26 and 34, 64; but MXFP4, 2880 x 2880, 128 experts 59, 70 and 55, 55, 64
// experts 50, 67 and 42, 54, 32 experts 39, 47 and 40, 40 (16 slots: 39, 34, 28 and 42, 39, 30), 16 experts 32, 35 and
// 40, 40.
bool moe_few(uint64_t n_slots, uint64_t n_expert, unsigned ty, unsigned ty2) {
    return n_slots <= MOEARC_MOE_SMALL_SLOTS && !(ty == 39u && ty2 == 39u && n_slots > 24 && n_expert >= 32);
}

// Groups a chunk's slots by expert, for weights of type ty, and ty2 in the product after it.
// x_n elements of x, for weights of type ty, are laid out for the matrix cores in the same launch; f16 ones of types
// whose order is the natural one are taken as they are.
int moe_plan(moearc_ctx *c, MoeArgs &a, const unsigned int *ids, uint32_t n_slots, uint32_t n_expert, bool half, unsigned ty,
             unsigned ty2, size_t x_n, uint8_t *ws, const MoeSpace &sp) {
    a.ids = ids;
    a.n_slots = n_slots;
    a.n_expert = n_expert;
    a.err = c->err_word;
    if (moe_few(n_slots, n_expert, ty, ty2)) return OK;
    MoePlanArgs p{};
    p.ids = ids;
    p.n_tiles = (uint32_t *) ws;
    p.tiles = (MoeTile *) (ws + sp.tiles);
    p.list = (uint32_t *) (ws + sp.list);
    p.err = c->err_word;
    p.n_slots = n_slots;
    p.n_expert = n_expert;
    p.tile = moe_light(n_slots, n_expert, half) ? MOEARC_MOE_LIGHT : MOEARC_MOE_TILE;
    a.tiles = p.tiles;
    a.n_tiles = p.n_tiles;
    a.list = p.list;
    if (half && (ty == 1u || ty == 8u)) return launch(c, c->f_moe_plan[2], n_expert + 1, 1024, p, nullptr, n_slots, n_expert, "moe_plan");
    p.prep.x = a.x;
    p.prep.hi = (uint16_t *) (ws + sp.split);
    p.prep.lo = p.prep.hi + sp.split_n;
    p.prep.n = x_n;
    p.prep.type = ty;
    a.x = p.prep.hi;
    a.x_lo = p.prep.lo;
    const unsigned blocks = (unsigned) std::min<size_t>((x_n / 8 + 1023) / 1024, 16384);
    return launch(c, c->f_moe_plan[half], n_expert + 1 + blocks, 1024, p, nullptr, n_slots, n_expert, "moe_plan");
}

// One grouped product (two matrices: gate, up and their activation). Without a plan x is as the caller's
// (f32, or f16 with `half`), with one always f16.
int moe_product(moearc_ctx *c, MoeArgs a, unsigned ty, bool gate_up, bool half) {
    const int i = moe_index(ty), g = gate_up ? 0 : 1;
    const char *const name = gate_up ? "moe_gate_up" : "moe_product";
    a.row_bytes = (uint64_t) a.cols / moearc_mv_be(ty) * moearc_mv_bb(ty);
    a.expert_bytes = a.row_bytes * a.rows;
    if (a.tiles) {
        const bool light = moe_light(a.n_slots, a.n_expert, half);
        const uint32_t per = moe_tile_rows(ty, half, light, gate_up);
        a.row_tiles = (a.rows + per - 1) / per;
        const uint64_t most = a.row_tiles * moe_max_tiles(a.n_slots, a.n_expert, light ? MOEARC_MOE_LIGHT : MOEARC_MOE_TILE);
        const unsigned grid = (unsigned) ((most + 7) / 8 * 8);  // eight runs, one per XCD
        return launch(c, (light ? c->f_moe_light : c->f_moe_tile)[i][g][half], grid, 256, a, nullptr, a.rows, a.n_slots, name);
    }
    const uint64_t nb = a.cols / 32, gran = (ty == 12u || ty == 13u || ty == 14u) ? 8 : 1;
    a.kb_per = (uint32_t) (((nb + MOEARC_MOE_SMALL_WAVES - 1) / MOEARC_MOE_SMALL_WAVES + gran - 1) / gran * gran);
    return launch2d(c, c->f_moe_small[i][g][half], (a.rows + (gate_up ? 15 : 31)) / (gate_up ? 16 : 32), a.n_slots,
                    64 * MOEARC_MOE_SMALL_WAVES, a, nullptr, a.rows, a.n_slots, 0, name);
}

// Whether a product of a single token's slots can run on moe_vec.hip: its row within one pass of a wave's lanes, its
// inputs in LDS beside the waves' buffers. Sets the launch's shape; rows_most: per wave, what its lanes can hold.
constexpr unsigned kMoeVecWaves = 8;
bool moe_vec_shape(MoeVecArgs &a, unsigned ty, unsigned n_rows_of_x, unsigned rows_most, unsigned &ppl, unsigned &lds) {
    const uint32_t pe = moearc_mv_pe(ty);
    a.n_pieces = (a.cols + pe - 1) / pe;
    if (a.n_pieces > 256) return false;
    ppl = a.n_pieces <= 64 ? 1 : a.n_pieces <= 128 ? 2 : 4;
    a.row_bytes = (uint64_t) a.cols / moearc_mv_be(ty) * moearc_mv_bb(ty);
    a.expert_bytes = a.row_bytes * a.rows;
    a.wave_buf = moearc_mv_wave_buf(a.row_bytes);
    a.x_lds_bytes = 4u * n_rows_of_x * a.n_pieces * (pe + 4u);
    lds = a.x_lds_bytes + kMoeVecWaves * a.wave_buf;
    // two work-groups per CU: a wave's rows share the inputs in its registers (one to four measured alike)
    const uint64_t slots = n_rows_of_x > 1 ? 1 : a.n_used, waves = 512ul * kMoeVecWaves;
    a.rpw = (uint32_t) std::min<uint64_t>(rows_most, (a.rows * slots + waves - 1) / waves);
    return lds <= 65536u && a.rpw > 0;
}

// One token's expert half, in two launches; ERR_ARG: another kernel's.
int moe_token(moearc_ctx *c, const moearc_moe *m, void *y, const void *x, bool half, const unsigned int *ids, const float *weights,
              unsigned long n_used, unsigned accumulate, uint8_t *act) {
    if (n_used > 64) return ERR_ARG;
    MoeVecArgs g{};
    g.ids = ids;
    g.weights = weights;
    g.err = c->err_word;
    g.n_used = (uint32_t) n_used;
    g.n_expert = (uint32_t) m->n_expert;
    g.x_f16 = g.y_f16 = half;
    MoeVecArgs d = g;
    unsigned gp, gl, dp, dl;
    g.rows = d.cols = (uint32_t) m->n_ff;
    g.cols = d.rows = (uint32_t) m->n_embd;
    if (!moe_vec_shape(g, m->w_type[0], 1, 32, gp, gl) || !moe_vec_shape(d, m->w_type[2], (unsigned) n_used, 64 / (unsigned) n_used, dp, dl))
        return ERR_ARG;
    for (int i = 0; i < 2; ++i) {
        g.w[i] = (const uint8_t *) m->w[i];
        g.bias[i] = m->bias[i];
    }
    g.x = x;
    g.y = act;
    g.clamped = m->act == MOEARC_ACT_SWIGLU_CLAMPED;
    g.alpha = m->alpha;
    g.limit = m->limit;
    d.w[0] = (const uint8_t *) m->w[2];
    d.bias[0] = m->bias[2];
    d.x = act;
    d.y = y;
    d.accumulate = accumulate;
    const unsigned per_g = kMoeVecWaves * g.rpw, per_d = kMoeVecWaves * d.rpw;
    auto form = [](unsigned ppl) { return ppl == 1 ? 0 : ppl == 2 ? 1 : 2; };
    if (const int rc = launch2d(c, c->f_moe_vec[moe_index(m->w_type[0])][0][form(gp)], (g.rows + per_g - 1) / per_g, (unsigned) n_used,
                                64 * kMoeVecWaves, g, nullptr, g.rows, n_used, gl, "moe_gate_up"))
        return rc;
    return launch2d(c, c->f_moe_vec[moe_index(m->w_type[2])][1][form(dp)], (d.rows + per_d - 1) / per_d, 1, 64 * kMoeVecWaves, d, nullptr,
                    d.rows, n_used, dl, "moe_down");
}

// Brackets a call of several launches under one key, as a single launch would be.
struct LaunchScope {
    moearc_ctx *c;
    const char *what;
    unsigned long r, m;
    hipEvent_t start = nullptr;
    LaunchScope(moearc_ctx *c, const char *what, unsigned long r, unsigned long m) : c(c), what(what), r(r), m(m) {
        if (tracks(c, what) && (start = take_event(c)) && hipEventRecord(start, c->stream) != hipSuccess) {
            c->event_pool.push_back(start);
            start = nullptr;
        }
        ++c->scope_depth;
    }
    ~LaunchScope() {
        --c->scope_depth;
        if (start) record_bracket(c, start, what, r, m);
    }
};

bool moe_load(moearc_ctx *c) {
    struct {
        hipFunction_t *slot;
        const char *name;
    } fns[] = {
        {&c->f_norm[0][0], "moearc_norm_r16_v1_k"},   {&c->f_norm[0][1], "moearc_norm_r16_v4_k"},
        {&c->f_norm[1][0], "moearc_norm_r64_v1_k"},   {&c->f_norm[1][1], "moearc_norm_r64_v4_k"},
        {&c->f_norm[2][0], "moearc_norm_r256_v1_k"},  {&c->f_norm[2][1], "moearc_norm_r256_v4_k"},
        {&c->f_norm[3][0], "moearc_norm_r1024_v1_k"}, {&c->f_norm[3][1], "moearc_norm_r1024_v4_k"},
        {&c->f_norm_long, "moearc_norm_long_k"},
        {&c->f_route[0], "moearc_moe_route_p1_k"},    {&c->f_route[1], "moearc_moe_route_p2_k"},
        {&c->f_route[2], "moearc_moe_route_p4_k"},    {&c->f_route[3], "moearc_moe_route_p8_k"},
        {&c->f_route[4], "moearc_moe_route_p16_k"},   {&c->f_route[5], "moearc_moe_route_p32_k"},
        {&c->f_route[6], "moearc_moe_route_p64_k"},   {&c->f_moe_plan[2], "moearc_moe_plan_k"},
        {&c->f_moe_plan[0], "moearc_moe_plan_f32_k"}, {&c->f_moe_plan[1], "moearc_moe_plan_f16_k"},
        {&c->f_moe_combine, "moearc_moe_combine_k"},
    };
    auto get = [&](hipFunction_t *slot, const char *name) {
        if (hipModuleGetFunction(slot, c->module, name) == hipSuccess) return true;
        std::fprintf(stderr, "moearc: code object lacks kernel %s\n", name);
        return false;
    };
    for (auto &f : fns)
        if (!get(f.slot, f.name)) return false;
    for (int t = 0; t < 6; ++t)
        for (int i = 0; i < 4; ++i) {
            char name[64];
            std::snprintf(name, sizeof(name), "moearc_moe_small_%s_%s_%s_k", kMoeNames[t], i & 2 ? "p" : "gu", i & 1 ? "f16" : "f32");
            if (!get(&c->f_moe_small[t][i >> 1][i & 1], name)) return false;
            if (i < 3) {  // gate and up, down x 1, 2, 4 pieces per lane
                for (int k = 0; k < 2; ++k) {
                    std::snprintf(name, sizeof(name), "moearc_moe_vec_%s_%s_p%d_k", kMoeNames[t], k ? "down" : "gu", 1 << i);
                    if (!get(&c->f_moe_vec[t][k][i], name)) return false;
                }
            }
            std::snprintf(name, sizeof(name), "moearc_moe_tile_%s_%s_%s_k", kMoeNames[t], i & 2 ? "p" : "gu", i & 1 ? "f16" : "f32");
            if (!get(&c->f_moe_tile[t][i >> 1][i & 1], name)) return false;
            std::snprintf(name, sizeof(name), "moearc_moe_light_%s_%s_%s_k", kMoeNames[t], i & 2 ? "p" : "gu", i & 1 ? "f16" : "f32");
            if (!get(&c->f_moe_light[t][i >> 1][i & 1], name)) return false;
        }
    return true;
}

}  // namespace

extern "C" {

int moearc_norm_residual(moearc_ctx *c, void *x, unsigned int x_type, float *h, const void *y, unsigned int y_type,
                         const float *w_post, const float *gate, unsigned long gate_stride, float scale,
                         const float *w_pre, unsigned long n_rows, unsigned long n_cols, float eps) {
    if (!c || !h || (!x && !y)) return ERR;
    if (x_type > MOEARC_OUT_F16 || y_type > MOEARC_OUT_F16 || (!y && (w_post || gate)) || (!x && w_pre) || n_cols == 0 ||
        n_cols >= 0x40000000ul || n_rows >= 0x80000000ul || (gate && gate_stride != 0 && gate_stride < n_cols) || !(eps >= 0.f))
        return ERR_ARG;
    if (n_rows == 0) return OK;
    NormArgs a{};
    a.x = x;
    a.h = h;
    a.y = y;
    a.w_post = w_post;
    a.gate = gate;
    a.w_pre = w_pre;
    a.gate_stride = gate_stride;
    a.n_rows = (uint32_t) n_rows;
    a.n_cols = (uint32_t) n_cols;
    a.scale = scale;
    a.eps = eps;
    a.x_f16 = x_type == MOEARC_OUT_F16;
    a.y_f16 = y_type == MOEARC_OUT_F16;
    // four floats at a time where every row allows
    const bool by4 = n_cols % 4 == 0 && gate_stride % 4 == 0 &&
                     ((uintptr_t) h | (uintptr_t) w_post | (uintptr_t) gate | (uintptr_t) w_pre) % 16 == 0 &&
                     (uintptr_t) x % (a.x_f16 ? 8 : 16) == 0 && (uintptr_t) y % (a.y_f16 ? 8 : 16) == 0;
    const int i = n_cols <= 16 * MOEARC_NORM_PER_THREAD ? 0 : n_cols <= 64 * MOEARC_NORM_PER_THREAD ? 1
                : n_cols <= 256 * MOEARC_NORM_PER_THREAD ? 2 : n_cols <= 1024 * MOEARC_NORM_PER_THREAD ? 3 : 4;
    const unsigned rows = i == 0 ? 16 : i == 1 ? 4 : 1, threads = i >= 3 ? 1024 : 256;
    const hipFunction_t f = i == 4 ? c->f_norm_long : c->f_norm[i][by4];
    const uint64_t most = kMaxThreads / threads * rows;  // rows of one launch
    if (n_rows <= most) return launch(c, f, (unsigned) ((n_rows + rows - 1) / rows), threads, a, "norm_residual", n_rows, n_cols);
    const LaunchScope scope(c, "norm_residual", n_rows, n_cols);
    for (uint64_t r = 0; r < n_rows; r += most) {
        a.n_rows = (uint32_t) std::min<uint64_t>(most, n_rows - r);
        if (const int rc = launch(c, f, (unsigned) ((a.n_rows + rows - 1) / rows), threads, a, nullptr, n_rows, n_cols, "norm_residual")) return rc;
        a.h += a.n_rows * n_cols;
        if (a.x) a.x = (uint8_t *) a.x + a.n_rows * n_cols * (a.x_f16 ? 2 : 4);
        if (a.y) a.y = (const uint8_t *) a.y + a.n_rows * n_cols * (a.y_f16 ? 2 : 4);
        if (a.gate) a.gate += a.n_rows * gate_stride;
    }
    return OK;
}

int moearc_moe_route(moearc_ctx *c, unsigned int *ids, float *weights, const float *logits, unsigned long n_tok,
                     unsigned long n_expert, unsigned long n_used, unsigned int mode, float scale) {
    if (!c || !ids || !weights || !logits) return ERR;
    if (n_expert == 0 || n_expert > MOEARC_MAX_EXPERTS || n_used == 0 || n_used > n_expert || n_tok >= 0x80000000ul ||
        mode > MOEARC_ROUTE_SOFTMAX_SELECTED)
        return ERR_ARG;
    if (n_tok == 0) return OK;
    RouteArgs a{logits, ids, weights, (uint32_t) n_tok, (uint32_t) n_expert, (uint32_t) n_used,
                      mode == MOEARC_ROUTE_SOFTMAX_ALL ? 1u : 0u, scale, 0u};
    int i = 0;
    while (((unsigned long) MOEARC_ROUTE_LANES << i) < n_expert) ++i;
    // a wave of four tokens per work-group while those leave compute units idle, else four waves
    const unsigned threads = n_tok <= 4096 ? 64 : 256, per = threads / MOEARC_ROUTE_LANES;
    const uint64_t most = kMaxThreads / MOEARC_ROUTE_LANES;  // tokens of one launch
    if (n_tok <= most) return launch(c, c->f_route[i], (unsigned) ((n_tok + per - 1) / per), threads, a, "moe_route", n_tok, n_expert);
    const LaunchScope scope(c, "moe_route", n_tok, n_expert);
    for (uint64_t t = 0; t < n_tok; t += most) {
        a.n_tok = (uint32_t) std::min<uint64_t>(most, n_tok - t);
        if (const int rc = launch(c, c->f_route[i], (a.n_tok + per - 1) / per, threads, a, nullptr, n_tok, n_expert, "moe_route")) return rc;
        a.logits += (uint64_t) a.n_tok * n_expert;
        a.ids += (uint64_t) a.n_tok * n_used;
        a.weights += (uint64_t) a.n_tok * n_used;
    }
    return OK;
}

int moearc_moe_workspace(unsigned long n_tok, unsigned long n_used, unsigned long n_expert, unsigned long n_embd,
                         unsigned long n_ff, unsigned long *bytes) {
    if (!bytes) return ERR;
    if (moe_count_check(n_tok, n_used, n_expert, 0) || !moe_cols_ok(n_embd) || (n_ff && !moe_cols_ok(n_ff)) ||
        !moe_ffn_fits(n_used, n_ff))
        return ERR_ARG;
    *bytes = moe_space(n_tok, n_used, n_expert, n_embd, n_ff, moe_ffn_chunk(n_used, n_embd, n_ff)).bytes;
    return OK;
}

int moearc_matmul_experts(moearc_ctx *c, unsigned int type_id, void *y, const void *w, const void *x, unsigned int io_type,
                          const float *bias, const unsigned int *ids, unsigned long n_tok, unsigned long n_used,
                          unsigned long n_expert, unsigned int x_per_slot, unsigned long n_rows, unsigned long n_cols,
                          void *ws, unsigned long ws_bytes) {
    if (!c || !y || !w || !x || !ids) return ERR;
    if (const int rc = moe_count_check(n_tok, n_used, n_expert, io_type)) return rc;
    if (const int rc = moe_matrix_check(type_id, w, n_rows, n_cols)) return rc;
    if (x_per_slot > 1) return ERR_ARG;
    const unsigned long chunk = moe_chunk(n_used, n_cols);
    const MoeSpace sp = moe_space(n_tok, n_used, n_expert, n_cols, 0, chunk);
    if (const int rc = moe_space_check(sp.bytes, ws, ws_bytes)) return rc;
    if (n_tok == 0) return OK;
    uint8_t *mem;
    if (const int rc = moe_take_space(c, sp.bytes, ws, &mem)) return rc;
    moe_arm(c, ws);
    const size_t elem = io_type == MOEARC_OUT_F16 ? 2 : 4;
    const LaunchScope scope(c, "matmul_experts", n_rows, n_tok * n_used);
    const unsigned long step = std::min<unsigned long>(chunk, moe_chunk(n_used, n_rows));  // (the workspace does not know n_rows)
    for (unsigned long t = 0; t < n_tok; t += step) {
        const unsigned long n = std::min(step, n_tok - t);
        MoeArgs a{};
        a.x = (const uint8_t *) x + (x_per_slot ? t * n_used : t) * n_cols * elem;
        a.x_div = x_per_slot ? 1u : (uint32_t) n_used;
        const bool half = io_type == MOEARC_OUT_F16;
        if (const int rc = moe_plan(c, a, ids + t * n_used, (uint32_t) (n * n_used), (uint32_t) n_expert, half, type_id, type_id,
                                    (x_per_slot ? n * n_used : n) * n_cols, mem, sp))
            return rc;
        a.w[0] = (const uint8_t *) w;
        a.bias[0] = bias;
        a.y = (uint8_t *) y + t * n_used * n_rows * elem;
        a.y_f16 = half;
        a.zero_skipped = 1u;
        a.rows = (uint32_t) n_rows;
        a.cols = (uint32_t) n_cols;
        if (const int rc = moe_product(c, a, type_id, false, half)) return rc;
    }
    return OK;
}

int moearc_moe_ffn(moearc_ctx *c, const moearc_moe *m, void *y, const void *x, unsigned int io_type, const unsigned int *ids,
                   const float *weights, unsigned long n_tok, unsigned long n_used, unsigned int accumulate, void *ws,
                   unsigned long ws_bytes) {
    if (!c || !m || !y || !x || !ids || !weights || !m->w[0] || !m->w[1] || !m->w[2]) return ERR;
    if (const int rc = moe_count_check(n_tok, n_used, m->n_expert, io_type)) return rc;
    if (m->w_type[0] != m->w_type[1] || m->act > MOEARC_ACT_SWIGLU_CLAMPED || accumulate > 1 ||
        (accumulate && io_type != MOEARC_OUT_F32) || (m->act == MOEARC_ACT_SWIGLU_CLAMPED && !(m->limit >= 0.f)) ||
        !moe_ffn_fits(n_used, m->n_ff))
        return ERR_ARG;
    for (int i = 0; i < 3; ++i)
        if (const int rc = moe_matrix_check(m->w_type[i], m->w[i], i < 2 ? m->n_ff : m->n_embd, i < 2 ? m->n_embd : m->n_ff))
            return rc;
    const unsigned long chunk = moe_ffn_chunk(n_used, m->n_embd, m->n_ff);
    const MoeSpace sp = moe_space(n_tok, n_used, m->n_expert, m->n_embd, m->n_ff, chunk);
    if (const int rc = moe_space_check(sp.bytes, ws, ws_bytes)) return rc;
    if (n_tok == 0) return OK;
    uint8_t *mem;
    if (const int rc = moe_take_space(c, sp.bytes, ws, &mem)) return rc;
    moe_arm(c, ws);
    const bool half = io_type == MOEARC_OUT_F16;
    const size_t elem = half ? 2 : 4;
    const LaunchScope scope(c, "moe_ffn", m->n_ff, n_tok * n_used);
    if (n_tok == 1) {
        const int rc = moe_token(c, m, y, x, half, ids, weights, n_used, accumulate, mem + sp.act);
        if (rc != ERR_ARG) return rc;
    }
    for (unsigned long t = 0; t < n_tok; t += chunk) {
        const unsigned long n = std::min(chunk, n_tok - t);
        MoeArgs a{};
        a.x = (const uint8_t *) x + t * m->n_embd * elem;
        if (const int rc = moe_plan(c, a, ids + t * n_used, (uint32_t) (n * n_used), (uint32_t) m->n_expert, half, m->w_type[0], m->w_type[2],
                                    n * m->n_embd, mem, sp))
            return rc;
        MoeArgs g = a, d = a;
        g.x_div = (uint32_t) n_used;
        for (int i = 0; i < 2; ++i) {
            g.w[i] = (const uint8_t *) m->w[i];
            g.bias[i] = m->bias[i];
        }
        g.y_order = m->w_type[2];
        g.y = mem + sp.act;
        g.y_lo = (uint16_t *) (mem + sp.act) + sp.act_n;
        d.x_lo = g.y_lo;
        // f16 calls round the activations once: hi + lo would double the down product's MFMAs and its reads of them, to
        // undo a rounding of the size that x came with
        g.y_f16 = half;
        g.rows = (uint32_t) m->n_ff;
        g.cols = (uint32_t) m->n_embd;
        g.clamped = m->act == MOEARC_ACT_SWIGLU_CLAMPED;
        g.alpha = m->alpha;
        g.limit = m->limit;
        if (const int rc = moe_product(c, g, m->w_type[0], true, half)) return rc;
        d.x = mem + sp.act;
        d.x_div = 1u;
        d.w[0] = (const uint8_t *) m->w[2];
        d.bias[0] = m->bias[2];
        d.y = mem + sp.part;
        d.rows = (uint32_t) m->n_embd;
        d.cols = (uint32_t) m->n_ff;
        if (const int rc = moe_product(c, d, m->w_type[2], false, half)) return rc;
        MoeCombineArgs s{};
        s.part = (const float *) (mem + sp.part);
        s.weights = weights + t * n_used;
        s.ids = ids + t * n_used;
        s.y = (uint8_t *) y + t * m->n_embd * elem;
        s.n_tok = (uint32_t) n;
        s.n_used = (uint32_t) n_used;
        s.n_expert = (uint32_t) m->n_expert;
        s.cols = (uint32_t) m->n_embd;
        s.y_f16 = half;
        s.accumulate = accumulate;
        if (const int rc = launch2d(c, c->f_moe_combine, (unsigned) ((m->n_embd / 4 + 255) / 256), (unsigned) n, 256, s, nullptr, n,
                                    m->n_embd, 0, "moe_combine"))
            return rc;
    }
    return OK;
}

}  // extern "C"
