// Attention of a ragged batch's new tokens over the paged f16 cache: sequences with any number of new
// tokens each (decode steps, drafts, prompt chunks), heads of up to 256 channels, any group and page size.
// Row (token i of n new ones, head) of a sequence with n_kv keys sits at p = n_kv - n + i and attends keys
// [max(0, p + 1 - n_swa), p] (n_swa 0: [0, p]) with the head's sink in the denominator; a row at p < 0 sees
// nothing and is zero.
//
// A work-group owns one KV head and a tile of rows, a row being a (token, head of the KV head's group) pair, so K and V
// are read once for all of a tile's heads. Full tiles have 128 rows, 32 to each of the four waves; keys stream through
// LDS in 32-key tiles, four buffers, copies (LDS DMA, 16 bytes a lane) three tiles ahead, one barrier a tile. Small
// tiles have 32 rows, which all waves hold, each with every fourth 32 keys in a buffer of its own, no barriers; the waves'
// sums meet in LDS at the end. Tiles whose keys are cut into pieces (few rows, many keys) leave records that the merge
// kernel joins. The host's plan chooses between these (batch_plan, with what each measured).
//
// Bounds and what whole calls measured on MI355X, in a long run of them (a 1 GiB copy there 5.12 TB/s, an 8192^3 f16 product
// 1.16 PFLOP/s):
//   full tiles, 128 channels: power; 512 tokens behind 32,700, 32 heads over 4: 299 us, 924 TFLOP/s, the matrix cores busy for
//     53% of the time at 1.73 GHz; 4096 tokens from the start 155 us, 886 TFLOP/s. Pages of no multiple of eight tokens: 361 and
//     187, since each lane's copy takes an address of its own instead of a wave's base
//   full tiles, 64 channels: the softmax's vector instructions, of which a score has as many beside half the products: four
//     prompts of 2048, 64 heads over 8: 198 us, 696 TFLOP/s
//   full tiles, 256 channels: one work-group a CU, so nobody's products run beside a wave's softmax; 512 tokens behind 16,000,
//     16 heads over 2: 217 us, 627 TFLOP/s; 4096 from the start 240 us, 573 TFLOP/s
//   decode steps beside prompt pieces, 32 sequences: HBM; 46.6 us for 166 MB, 3.6 TB/s, and 5.5 for the merge
//   few tokens: latency, a trip to the block table, to the keys, and the merge's launch; 18 tokens of four drafts 13.7 us
//
// Matrix layout (v_mfma_f32_32x32x16_f16, DB = channels / 32):
//   S^T[32 keys x 32 rows] = K . Q^T          2 DB MFMAs
//   O^T[32 DB ch x 32 rows] += V^T . P^T      2 DB MFMAs
// Lane (h, n) = (lane / 32, lane % 32) holds S^T rows 8j + 4h + i (j, i = 0..3) of column n, sixteen keys of query row
// n, in the order in which P^T's operand wants them (keys 16s + 4h + i and 16s + 8 + 4h + i of step s): the weights
// go from one product into the next in registers, and a row's statistics are one lane pair's.
//
// LDS rows are 64 DB bytes, 16-byte chunks c XOR-swizzled by the key k so that every pass of a read touches each bank
// once (256 bytes a clock; a b128 read is served sixteen lanes i..i+7, i+16..i+23 at a time, a transposing b64 read 32):
//   K: c ^ f(k), f = (k & 7) ^ (k >> 4 & 1) at DB 2 (two rows to 256 bytes), (k & 7) | (k >> 4 & 1) << 3 above
//   V: c ^ f(k), f = (k & 7) ^ (k >> 1 & 1) << 2 at DB 2, (k & 3) << 2 above
//
// Softmax in the log2 domain against a row reference m that moves only when a weight leaves f16's range (a score
// more than 9 above m), as prefill.hip explains. Default kernels round a weight to f16 once (at most 2^-11 of it,
// the row sum is over the rounded ones; that is half of what rounding the output to f16 costs, and less after
// averaging); precise ones, for f32 outputs, carry it as f16 hi + lo (2^-22).
//
// Infinities and NaN in V of keys that a row does not see must not reach it, but 0 * NaN would in the matrix cores.
// A work-group that ends with a non-finite accumulator runs once more, with the tiles that cross a mask done key by key and
// without the chunks behind a narrower head's channels.
#include "common.h"

namespace {

template <int DB>
struct AbShape {
    static constexpr uint32_t ROW = 64u * DB;        // bytes of a key's row in LDS
    static constexpr uint32_t CHUNKS = 4u * DB;      // of 16 bytes
    static constexpr uint32_t TILE = 32u * ROW;      // one K or V tile
    static constexpr uint32_t BUF = 2u * TILE;
    static constexpr uint32_t KEYS = 64u / CHUNKS;   // keys that one copy instruction of a wave fills
    static constexpr uint32_t COPIES = 8u / KEYS;    // instructions a wave gives each of K and V per tile (8 keys)
    static __device__ __forceinline__ uint32_t fk(uint32_t k) {
        return DB == 2 ? (k & 7u) ^ ((k >> 4) & 1u) : (k & 7u) | ((k >> 4) & 1u) << 3;
    }
    static __device__ __forceinline__ uint32_t fv(uint32_t k) {
        return DB == 2 ? (k & 7u) ^ ((k >> 1) & 1u) << 2 : (k & 3u) << 2;
    }
    static __device__ __forceinline__ uint32_t k_at(uint32_t k, uint32_t c) { return k * ROW + ((c ^ fk(k)) << 4); }
    static __device__ __forceinline__ uint32_t v_at(uint32_t k, uint32_t c) { return k * ROW + ((c ^ fv(k)) << 4); }
};

typedef short short4v_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v_t lds_short4_t;
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;

// LDS DMA of 16 bytes per lane to LDS address lds + 16 * lane, from a lane's own address, or from wave-uniform ones of K
// and V plus a lane's offsets: COPIES times, 1 KB of LDS apart, V's `v_lds` behind K's. Through asm: for the builtin the
// compiler, which cannot tell the buffer being read from the one being filled, would wait for the copy before every LDS
// read. One statement for a tile's copies: m0 (the LDS address; the compiler's) is saved and restored once. A wave issues
// one instruction in four cycles, so every scalar one that the key loop is spared counts.
__device__ __forceinline__ void ab_copy16(const uint8_t *p, uint32_t lds) {
    uint32_t m0_saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t"
                 "s_mov_b32 m0, %0"
                 : "=&s"(m0_saved) : "v"(p), "s"(lds) : "memory");
}
#define AB_NEXT "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 "
template <int COPIES>
__device__ __forceinline__ void ab_copy(const uint8_t *base, const uint32_t (&off)[COPIES], uint32_t lds) {
    uint32_t m0_saved;
    if constexpr (COPIES == 1)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %2\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(m0_saved) : "s"(lds), "s"(base), "v"(off[0]) : "memory");
    else if constexpr (COPIES == 2)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %2\n\t"
                     AB_NEXT "%4, %2\n\ts_mov_b32 m0, %0"
                     : "=&s"(m0_saved) : "s"(lds), "s"(base), "v"(off[0]), "v"(off[1]) : "memory", "scc");
    else
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %2\n\t"
                     AB_NEXT "%4, %2\n\t" AB_NEXT "%5, %2\n\t" AB_NEXT "%6, %2\n\ts_mov_b32 m0, %0"
                     : "=&s"(m0_saved)
                     : "s"(lds), "s"(base), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]) : "memory", "scc");
}
template <int COPIES>
__device__ __forceinline__ void ab_copy_kv(const uint8_t *k, const uint8_t *v, const uint32_t (&ok)[COPIES],
                                           const uint32_t (&ov)[COPIES], uint32_t k_lds, uint32_t v_lds) {
    uint32_t m0_saved;
    if constexpr (COPIES == 1) {
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %3\n\t"
                     "s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %6, %4\n\ts_mov_b32 m0, %0"
                     : "=&s"(m0_saved) : "s"(k_lds), "s"(v_lds), "s"(k), "s"(v), "v"(ok[0]), "v"(ov[0]) : "memory");
    } else if constexpr (COPIES == 2) {
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %3\n\t"
                     AB_NEXT "%6, %3\n\t"
                     "s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %7, %4\n\t"
                     AB_NEXT "%8, %4\n\ts_mov_b32 m0, %0"
                     : "=&s"(m0_saved)
                     : "s"(k_lds), "s"(v_lds), "s"(k), "s"(v), "v"(ok[0]), "v"(ok[1]), "v"(ov[0]), "v"(ov[1])
                     : "memory", "scc");
    } else {
        ab_copy<COPIES>(k, ok, k_lds);
        ab_copy<COPIES>(v, ov, v_lds);
    }
}
#undef AB_NEXT

// The slot whose work items (begin[] ascending, entries n .. the end: the count) hold `item`.
__device__ __forceinline__ uint32_t ab_slot(const uint32_t *begin, uint32_t item) {
    uint32_t g = 0;
#pragma unroll
    for (uint32_t i = 1; i < MOEARC_BATCH_SEQS / 8; ++i) g += item >= begin[8 * i];
    uint32_t b = 8 * g;
#pragma unroll
    for (uint32_t i = 1; i < 8; ++i) b += item >= begin[8 * g + i];
    return b;
}

// x / group for x < 2^31 (the host's factor and shift).
__device__ __forceinline__ uint32_t ab_token(const AttnBatchArgs &a, uint32_t x) {
    return (uint32_t) ((uint64_t) x * a.group_magic >> a.group_shift);
}

// Keys [lo, hi) that the rows of tile t (of tile_rows) of a slot see. No other's block-table entry is looked at.
struct AbSpan {
    uint32_t lo, hi;
};
__device__ __forceinline__ AbSpan ab_span(const AttnBatchArgs &a, uint32_t n, uint32_t n_kv, uint32_t t, uint32_t tile_rows) {
    const int32_t shift = (int32_t) (n_kv - n);  // a token's position less its index; below 0: the first see nothing
    const uint32_t tok0 = ab_token(a, t * tile_rows), tok1 = min(ab_token(a, t * tile_rows + tile_rows - 1u), n - 1u);
    const int32_t last = shift + (int32_t) tok1, first = max(0, shift + (int32_t) tok0);
    AbSpan s;
    s.hi = last < 0 ? 0u : (uint32_t) last + 1u;
    s.lo = a.n_swa && (uint32_t) first + 1u > a.n_swa ? (uint32_t) first + 1u - a.n_swa : 0u;
    if (a.eights) s.lo &= ~7u;  // in the same page
    return s;
}

// A head's sink in the log2 domain. Above 2.3e38 the product overflows, and inf - inf would make NaN of a row that is zero.
__device__ __forceinline__ float ab_sink(float sink) { return fminf(sink * MOEARC_LOG2E, 3.0e38f); }

// A wave-uniform value that is there from here on: arguments are loaded together at a kernel's start, where the compiler
// would put each in front of its first use, a chain of waits.
#define AB_HERE(x) asm volatile("" : "+s"(x))

template <int DB, bool PRECISE>
__device__ __forceinline__ void ab_body(const AttnBatchArgs &a) {
    using S = AbShape<DB>;
    constexpr uint32_t NBUF = 4, COPIES = S::COPIES;
    __shared__ __attribute__((aligned(1024))) uint8_t tiles[NBUF * S::BUF];
    __shared__ uint32_t table[MOEARC_AB_PT + 4];  // places in the pools (page * page_tokens + slot) of eight keys each, or of each key
    uint32_t *const again = table + MOEARC_AB_PT;  // the waves' votes

    const uint32_t tid = threadIdx.x, lane = tid & 63u, h = lane >> 5, n = lane & 31u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t G = a.n_kv_heads, kv_magic = a.kv_magic, kv_shift = a.kv_shift, n_slots = a.n_slots, n_heads = a.n_heads;
    uint32_t D = a.head_dim, group = a.group, n_swa = a.n_swa, page_tokens = a.page_tokens, n_pages = a.n_pages;
    const uint16_t *q_base = a.q;
    const uint8_t *k_pool = (const uint8_t *) a.k_pages, *v_pool = (const uint8_t *) a.v_pages;
    const float *sinks = a.sinks;
    const uint32_t *row_table = a.block_tables;
    uint64_t bt_stride = a.bt_stride;
    AB_HERE(G); AB_HERE(kv_magic); AB_HERE(kv_shift); AB_HERE(n_slots); AB_HERE(n_heads); AB_HERE(D); AB_HERE(group); AB_HERE(n_swa);
    AB_HERE(page_tokens); AB_HERE(n_pages); AB_HERE(q_base); AB_HERE(k_pool); AB_HERE(v_pool); AB_HERE(sinks); AB_HERE(row_table);
    AB_HERE(bt_stride);
    const uint32_t item = (uint32_t) ((uint64_t) blockIdx.x * kv_magic >> kv_shift), kvh = blockIdx.x - item * G;
    const uint32_t b = n_slots > 1u ? ab_slot(a.item_begin, item) : 0u;
    uint32_t n_new = a.slot[b].n_new, nt = a.slot[b].n_tiles, item0 = a.slot[b].item_begin, n_kv = a.slot[b].n_kv;
    uint32_t seq = a.slot[b].seq, tok_row = a.slot[b].row0, pieces = a.slot[b].pieces, piece = a.slot[b].piece;
    uint32_t tile_rows = a.slot[b].tile_rows;
    AB_HERE(n_new); AB_HERE(nt); AB_HERE(item0); AB_HERE(n_kv); AB_HERE(seq); AB_HERE(tok_row); AB_HERE(pieces); AB_HERE(piece);
    AB_HERE(tile_rows);
    const uint32_t rows = n_new * group, in_slot = item - item0;
    const bool few = tile_rows == 32u;  // the four waves share the rows, each with keys of its own
    const uint32_t pc = pieces > 1u ? in_slot / nt : 0u;
    const uint32_t tile = nt - 1u - (in_slot - pc * nt);  // the latest tile, which has the most keys, first
    const AbSpan span = ab_span(a, n_new, n_kv, tile, tile_rows);
    const uint32_t lo = span.lo + pc * piece;  // with pages of eights a multiple of 8
    const uint32_t hi = pieces > 1 ? min(span.hi, lo + piece) : span.hi;
    if (pc && lo >= span.hi) return;  // an earlier tile's span has fewer pieces
    row_table += seq * bt_stride;

    // ---- this lane's query row (rows behind the last are that one, and not stored) -------------------
    const int32_t shift = (int32_t) (n_kv - n_new);
    const uint32_t row0 = tile * tile_rows + (few ? 0u : wave * 32u), row = row0 + n;
    const bool row_ok = row < rows;
    const uint32_t tok = ab_token(a, min(row, rows - 1u)), hd = kvh * group + min(row, rows - 1u) - tok * group;
    const int32_t pos = shift + (int32_t) tok;
    // visible keys j: j - row_lo <= row_len as unsigned numbers (an empty row: at 2^31, which no key has)
    const uint32_t row_lo = pos < 0 ? 0x80000000u : n_swa && (uint32_t) pos + 1u > n_swa ? (uint32_t) pos + 1u - n_swa : 0u;
    const uint32_t row_len = pos < 0 ? 0u : (uint32_t) pos - row_lo;
    half8_t qop[2 * DB];
    {
        const uint16_t *q_row = q_base + (((uint64_t) tok_row + tok) * n_heads + hd) * D;
#pragma unroll
        for (int t = 0; t < 2 * DB; ++t)  // chunks behind the head's channels: any, for now
            qop[t] = __builtin_bit_cast(half8_t, *(const u32x4_t *) (q_row + min(16u * t + 8u * h, D - 8u)));
    }
    float c = a.scale_log2e;
    // positions of the wave's first and last row: which tiles cross a mask
    const int32_t w_first = shift + (int32_t) ab_token(a, min(row0, rows - 1u));
    const int32_t w_last = shift + (int32_t) ab_token(a, min(row0 + 31u, rows - 1u));
    const int32_t w_lo_last = n_swa ? max(0, w_last + 1 - (int32_t) n_swa) : 0;

    // ---- LDS addresses and copies ----------------------------------------------------------------
    uint32_t v_at[DB];
    {
        const uint32_t r = lane & 15u, q = (lane >> 4) & 1u, vkey = 4u * h + (r >> 2);
#pragma unroll
        for (int mb = 0; mb < DB; ++mb)
            v_at[mb] = S::TILE + S::v_at(vkey, 4u * mb + 2u * q + ((r >> 1) & 1u)) + ((r & 1u) << 3);
    }
    const uint32_t k_at = S::k_at(n, h);  // of MFMA t: ^ t << 5
    const uint32_t lds0 = (uint32_t) (uintptr_t) (lds_u8_t *) tiles;
    const uint32_t ld_key = lane / S::CHUNKS, ld_slot = lane % S::CHUNKS;  // of a copy's KEYS keys, and where in their rows
    const uint32_t key_bytes = G * D * 2u, head_bytes = kvh * D * 2u;
    const bool eights = a.eights;
    // What this lane copies of eight keys of K or V: byte offsets from their first one's row in the pool. The swizzle of eight
    // keys is one of two for K (by their bit 4), the same for all of V. Where a head has fewer channels than 32 DB, chunks
    // behind them are its first one again: q is zero there, and nobody stores what becomes of V's.
    struct Lanes {
        uint32_t off[COPIES];
    };
    auto lanes_of = [&](auto swizzle, uint32_t first) {
        Lanes l;
#pragma unroll
        for (uint32_t i = 0; i < COPIES; ++i) {
            const uint32_t key = ld_key + i * S::KEYS, ch = ld_slot ^ swizzle(first + key);
            l.off[i] = key * key_bytes + head_bytes + (8u * ch < D ? 16u * ch : 0u);
        }
        return l;
    };
    auto k_lanes = [&](uint32_t first) { return lanes_of([](uint32_t k) { return S::fk(k); }, first); };
    const Lanes v_lanes = lanes_of([](uint32_t k) { return S::fv(k); }, 0u);

    // Keys whose places fit `table` at a time (a segment); every thread of the work-group takes part. A segment is whole tiles:
    // masks go by what a row sees, so a tile's columns behind the segment's end would count, and again in the next one.
    static_assert(MOEARC_AB_PT % 32u == 0u, "a segment of whole tiles");
    const uint32_t seg_keys = eights ? 8u * MOEARC_AB_PT : MOEARC_AB_PT;
    bool again_round = false;
    auto load_places = [&](uint32_t seg, uint32_t last_key) {
        const uint32_t n_places = eights ? (last_key - seg) / 8u + 1u : last_key - seg + 1u;
        for (uint32_t i = tid; i < n_places; i += 256u) {
            const uint32_t key = seg + (eights ? 8u * i : i);
            const uint32_t page = (uint32_t) ((uint64_t) key * a.page_magic >> a.page_shift);
            uint32_t id = row_table[page];
            if (id >= n_pages) {  // reported; what is read instead lies in the pool
                *(volatile uint32_t *) a.err = 1u;
                id = 0u;
            }
            table[i] = id * page_tokens + (key - page * page_tokens);
        }
        __syncthreads();
    };
    auto next_places = [&](uint32_t seg, uint32_t last_key) {  // of a later segment, or the first again
        if (seg == lo && !again_round) return;
        __syncthreads();
        load_places(seg, last_key);
    };
    float sink2 = -INFINITY;
    if (sinks) sink2 = sinks[hd];
    if (lo < hi) load_places(lo, min(hi, lo + seg_keys) - 1u);
    // q has arrived here: the compiler would wait for its loads in the key loop, and so for the copies issued after them
#pragma unroll
    for (int t = 0; t < 2 * DB; ++t) {
        if (D < 32u * DB && 16u * t + 8u * h >= D) qop[t] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
        if (c < 0.f) qop[t] = -qop[t];  // s * c = (-s) * (-c): then the row maximum of s * c is c times the maximum of s
        if (c == 0.f) qop[t] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};  // every score 0, and masked ones still -inf
        asm volatile("" : "+v"(qop[t]));
    }
    c = c == 0.f ? 1.f : fabsf(c);
    sink2 = ab_sink(sink2);

    // Copies of eight keys: with pages of eights these share a page, and their base is wave-uniform; otherwise a lane looks
    // for its own key. Keys behind the last are that one: their scores are masked, and no slot is read that the cache has
    // not written.
    auto offset_of = [&](uint32_t place) { return (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) place) * key_bytes; };
    auto copy8_any = [&](const uint8_t *pool, const Lanes &l, uint32_t j, uint32_t seg, uint32_t last_key, uint32_t dst) {
#pragma unroll
        for (uint32_t i = 0; i < COPIES; ++i) {
            uint32_t off = l.off[i];
            asm volatile("" : "+v"(off));  // computed here: the loop that hardly takes this path has no registers for it
            const uint32_t key = ld_key + i * S::KEYS, at = min(j + key, last_key) - seg;
            const uint32_t place = eights ? table[at / 8u] + at % 8u : table[at];
            ab_copy16(pool + ((uint64_t) place * key_bytes + (off - key * key_bytes)), dst + i * 1024u);
        }
    };

    // ---- a tile's arithmetic -----------------------------------------------------------------------
    float m_run, l_run;
    float16_t O[DB];
    const half2_t ones2 = {1, 1};
    auto start = [&]() {
        m_run = PF_M_INIT;
        l_run = 0.f;
#pragma unroll
        for (int mb = 0; mb < DB; ++mb)
#pragma unroll
            for (int i = 0; i < 16; ++i) O[mb][i] = 0.f;
    };
    // S^T of the tile at kt. Chunks of K behind the head's channels hold its first one again: 0 * inf there is a NaN, which
    // makes the row's accumulators one, so the second run leaves these chunks out.
    auto scores = [&](auto by_key_c, const uint8_t *kt) {
        float16_t s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * DB; ++t) {
            half8_t k = *(const half8_t *) (kt + (k_at ^ (uint32_t) t << 5));
            if constexpr (decltype(by_key_c)::value)
                if (16u * t + 8u * h >= D) k = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
            s = pf_mfma(k, qop[t], s);
        }
        return s;
    };
    auto weights = [&](const float16_t &s, float bias, float l, half8_t (&phi)[2], half8_t (&plo)[2]) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i], c, bias)), p1 = __builtin_amdgcn_exp2f(fmaf(s[i + 1], c, bias));
            const half2_t hv = {(_Float16) p0, (_Float16) p1};
            phi[i >> 3][i & 7] = hv[0];
            phi[i >> 3][(i & 7) + 1] = hv[1];
            l = __builtin_amdgcn_fdot2(hv, ones2, l, false);
            if constexpr (PRECISE) {
                plo[i >> 3][i & 7] = (_Float16) (p0 - (float) hv[0]);
                plo[i >> 3][(i & 7) + 1] = (_Float16) (p1 - (float) hv[1]);
            }
        }
        return l;
    };
    // Whether a mask of some row of the wave lies in the tile of keys j0 .., and -inf for what a row does not see.
    auto crosses = [&](uint32_t j0) { return (int32_t) j0 + 31 > w_first || (int32_t) j0 < w_lo_last; };
    auto mask = [&](float16_t &s, uint32_t j0) {
        const uint32_t off = j0 + 4u * h - row_lo;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (off + (uint32_t) (8 * (i >> 2) + (i & 3)) > row_len) s[i] = -INFINITY;
    };
    auto add_lo = [&](float l, const half8_t (&plo)[2]) {
        if constexpr (PRECISE) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2((half2_t){plo[q][i], plo[q][i + 1]}, ones2, l, false);
        }
        return l;
    };
    auto overflow = [&](float l) { return __builtin_amdgcn_ballot_w64(l == INFINITY) != 0; };
    // The reference at the row's maximum with these scores.
    auto rescale = [&](const float16_t &s) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        top *= c;
        const float m_new = fmaxf(m_run, fmaxf(top, __shfl_xor(top, 32)));
        const float corr = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= corr;
#pragma unroll
        for (int mb = 0; mb < DB; ++mb) O[mb] *= corr;
    };
    // V^T's operand of channel block mb, step q; the product with the weights.
    auto operand = [&](const uint8_t *kt, int mb, int q) {
        const uint8_t *p = kt + v_at[mb] + q * 16 * S::ROW;
        const short4v_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t *) p);
        const short4v_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t *) (p + 8 * S::ROW));
        typedef short short8v_t __attribute__((ext_vector_type(8)));
        const short8v_t x = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(half8_t, x);
    };
    auto values = [&](const uint8_t *kt, const half8_t (&phi)[2], const half8_t (&plo)[2]) {
#pragma unroll
        for (int mb = 0; mb < DB; ++mb)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const half8_t va = operand(kt, mb, q);
                O[mb] = pf_mfma(va, phi[q], O[mb]);
                if constexpr (PRECISE) O[mb] = pf_mfma(va, plo[q], O[mb]);
            }
    };
    // The same key by key: weight and visibility from the lane that holds them.
    auto values_by_key = [&](const uint8_t *kt, uint32_t j0, const half8_t (&phi)[2], const half8_t (&plo)[2]) {
        for (uint32_t k = 0; k < 32u; ++k) {
            const uint32_t i = 4u * (k >> 3) + (k & 3u);  // register of lane half (k >> 2) & 1
            float w = 0.f;
#pragma unroll
            for (uint32_t r = 0; r < 16u; ++r)
                if (r == i) w = (float) phi[r >> 3][r & 7] + (PRECISE ? (float) plo[r >> 3][r & 7] : 0.f);
            w = __shfl(w, (int) (n + 32u * ((k >> 2) & 1u)));
            const bool sees = j0 + k - row_lo <= row_len;
#pragma unroll
            for (int mb = 0; mb < DB; ++mb) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t ch = 32u * mb + 8u * (r >> 2) + 4u * h + (r & 3u);
                    const float v = (float) *(const _Float16 *) (kt + S::TILE + S::v_at(k, ch >> 3) + 2u * (ch & 7u));
                    if (sees) O[mb][r] = fmaf(w, v, O[mb][r]);
                }
                asm volatile("" : : : "memory");  // sixteen values in flight
            }
        }
    };
    // A tile's weights and values, whatever happens in it; before_v() sees that V is there.
    auto absorb = [&](auto by_key_c, const float16_t &s, uint32_t j0, const uint8_t *kt, auto before_v) {
        half8_t phi[2], plo[2];
        float l = weights(s, MOEARC_AB_LOG2_PSCALE - m_run, l_run, phi, plo);
        if (overflow(l)) {
            rescale(s);
            l = weights(s, MOEARC_AB_LOG2_PSCALE - m_run, l_run, phi, plo);
        }
        l_run = add_lo(l, plo);
        before_v();
        if (decltype(by_key_c)::value && crosses(j0)) values_by_key(kt, j0, phi, plo);
        else values(kt, phi, plo);
    };
    auto any_not_finite = [&]() {
        bool finite = true;
        if (row_ok) {
#pragma unroll
            for (int mb = 0; mb < DB; ++mb)
#pragma unroll
                for (int i = 0; i < 16; ++i) finite = finite && (__float_as_uint(O[mb][i]) & 0x7F800000u) != 0x7F800000u;
        }
        const bool bad = __builtin_amdgcn_ballot_w64(!finite) != 0;
        if (lane == 0) again[wave] = bad;
        __syncthreads();
        return (again[0] | again[1] | again[2] | again[3]) != 0u;
    };

    // ---- the work-group's keys, all waves on the same 32 at a time -----------------------------------
    auto together = [&](auto by_key_c) {
        start();
        const Lanes k_own = k_lanes(8u * wave);
        for (uint32_t seg = lo; seg < hi; seg += seg_keys) {
            const uint32_t seg_hi = min(hi, seg + seg_keys), last_key = seg_hi - 1u;
            next_places(seg, last_key);
            // a wave's copies of a tile: eight keys of K and of V
            auto place_of = [&](uint32_t j0) { return eights ? table[(min(j0 + 8u * wave, last_key) - seg) / 8u] : 0u; };
            const uint32_t lds_own = __builtin_amdgcn_readfirstlane(lds0 + 8u * wave * S::ROW);
            auto copy_tile = [&](uint32_t j0, uint32_t buf, uint32_t place) {
                const uint32_t j = j0 + 8u * wave, dst = lds_own + buf * S::BUF;
                if (eights && j + 7u <= last_key) {
                    const uint64_t o = offset_of(place);
                    ab_copy_kv<COPIES>(k_pool + o, v_pool + o, k_own.off, v_lanes.off, dst, dst + S::TILE);
                } else {
                    copy8_any(k_pool, k_own, j, seg, last_key, dst);
                    copy8_any(v_pool, v_lanes, j, seg, last_key, dst + S::TILE);
                }
            };
            // Step r: this wave's copies of tile r + 1 are done (those of r + 2, issued later, may be in flight), every
            // wave meets, so all copies of r + 1 are in and nobody reads tile r - 1's buffer, which r + 3 then takes. Behind the
            // last tile there is nothing to wait for, and the scores beside the last weights are nobody's.
            const uint32_t steps = (seg_hi - seg + 31u) / 32u;
            auto first_key = [&](uint32_t r) { return seg + 32u * r; };
            constexpr int ONE = 2 * COPIES;  // a tile's copies
#pragma unroll 1
            for (uint32_t r = 0; r < min(steps, NBUF - 1u); ++r) copy_tile(first_key(r), r, place_of(first_key(r)));
            uint32_t ahead = steps >= NBUF ? place_of(first_key(NBUF - 1)) : 0u;  // read a step before its use
            if (steps > 2u) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * ONE) : "memory");
            else if (steps > 1u) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(ONE) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
            float16_t s = scores(by_key_c, tiles), next;
            auto open = [&](uint32_t r, uint32_t buf) {  // of tile r + 3
                if (r + 2u < steps) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(ONE) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
                if (r + NBUF - 1u < steps) {
                    copy_tile(first_key(r + NBUF - 1u), buf, ahead);
                    if (r + NBUF < steps) ahead = place_of(first_key(r + NBUF));
                }
            };
            for (uint32_t r = 0; r < steps; ++r) {
                open(r, (r + NBUF - 1u) % NBUF);
                if (crosses(first_key(r))) mask(s, first_key(r));
                next = scores(by_key_c, tiles + (r + 1u) % NBUF * S::BUF);  // beside the weights of this one
                absorb(by_key_c, s, first_key(r), tiles + r % NBUF * S::BUF, [] {});
                s = next;
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");  // before the buffers are filled again, or released
        }
    };
    // ---- few rows: each wave has every fourth 32 keys, in a buffer of its own ------------------------
    // No barriers: K's half is filled with the wave's next tile while the weights and V's product run, V's while the next
    // scores do. Eight waves of a CU keep 64 to 128 KB in flight.
    uint8_t *const own = tiles + wave * S::BUF;
    auto apart = [&](auto by_key_c) {
        start();
        const Lanes k0 = k_lanes(0u), k1 = k_lanes(16u);
        for (uint32_t seg = lo; seg < hi; seg += seg_keys) {
            const uint32_t seg_hi = min(hi, seg + seg_keys), last_key = seg_hi - 1u;
            next_places(seg, last_key);
            const uint32_t lds = __builtin_amdgcn_readfirstlane(lds0 + wave * S::BUF);
            auto copy32 = [&](const uint8_t *pages, const Lanes &l0, const Lanes &l1, uint32_t j, uint32_t dst) {
                if (eights && j + 31u <= last_key) {
#pragma unroll
                    for (uint32_t g = 0; g < 4u; ++g)
                        ab_copy<COPIES>(pages + offset_of(table[(j - seg) / 8u + g]), g < 2u ? l0.off : l1.off, dst + 8u * g * S::ROW);
                } else {
#pragma unroll 1
                    for (uint32_t g = 0; g < 2u; ++g) copy8_any(pages, l0, j + 8u * g, seg, last_key, dst + 8u * g * S::ROW);
#pragma unroll 1
                    for (uint32_t g = 2; g < 4u; ++g) copy8_any(pages, l1, j + 8u * g, seg, last_key, dst + 8u * g * S::ROW);
                }
            };
            auto copy_k = [&](uint32_t j) { copy32(k_pool, k0, k1, j, lds); };
            auto copy_v = [&](uint32_t j) { copy32(v_pool, v_lanes, v_lanes, j, lds + S::TILE); };
            uint32_t j0 = seg + 32u * wave;
            if (j0 < seg_hi) {
                copy_k(j0);
                copy_v(j0);
            }
            for (; j0 < seg_hi; j0 += 128u) {
                const bool more = j0 + 128u < seg_hi;
                asm volatile("s_waitcnt vmcnt(%0)" : : "n"(4 * COPIES) : "memory");  // V's may be in flight
                float16_t s = scores(by_key_c, own);
                asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // K has been read
                if (more) copy_k(j0 + 128u);
                if (crosses(j0)) mask(s, j0);
                absorb(by_key_c, s, j0, own, [&] {
                    if (more) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(4 * COPIES) : "memory");  // the next K's may be in flight
                    else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
                });
                asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // V has been read
                if (more) copy_v(j0 + 128u);
            }
        }
    };
    const uint64_t rec = ((uint64_t) a.slot[b].rec_begin + (tile * pieces + pc) * tile_rows) * G + kvh * tile_rows;  // row 0's record
    // Channels d .. d + 3 of out row `to`.
    auto store = [&](uint64_t to, uint32_t d, const float4_t &v) {
        if (a.out_f16) {
            const half2_t h0 = {(_Float16) v[0], (_Float16) v[1]}, h1 = {(_Float16) v[2], (_Float16) v[3]};
            *(u32x2_t *) ((_Float16 *) a.out + to * D + d) = u32x2_t{__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1)};
        } else {
            *(float4_t *) ((float *) a.out + to * D + d) = v;
        }
    };
    // 1 / (the row's sum with its sink), in the frame of m.
    auto inverse = [&](float m, float sum, float sink2) {
        const float top = fmaxf(m, sink2), f = __builtin_amdgcn_exp2f(m - top);
        const float total = sum * f + __builtin_amdgcn_exp2f(sink2 - top + MOEARC_AB_LOG2_PSCALE);
        return total == 0.f ? 0.f : f / total;  // a row without keys and without a sink
    };

    if (few) {
        apart(std::false_type{});
        again_round = any_not_finite();
        if (again_round) apart(std::true_type{});
        // the four waves' sums and outputs meet in LDS: row n's quad d / 4 at (d / 4) ^ (n & 7) of its 32 DB floats
        const float L = l_run + __shfl_xor(l_run, 32);
        float2_t *const ml = (float2_t *) table;
        __syncthreads();  // (with the places read)
        if (h == 0) ml[wave * 32u + n] = float2_t{m_run, L};
        if (tid < 32u) ml[128u + tid] = float2_t{sink2, 0.f};
#pragma unroll
        for (int mb = 0; mb < DB; ++mb)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                ((float4_t *) own)[n * 8u * DB + ((8u * mb + 2u * j + h) ^ (n & 7u))] =
                    float4_t{O[mb][4 * j], O[mb][4 * j + 1], O[mb][4 * j + 2], O[mb][4 * j + 3]};
        __syncthreads();
        const uint32_t r = tid >> 3, rr = tile * 32u + r;  // eight threads to a row
        if (rr >= rows) return;
        float m = ml[r][0], f[4], sum = 0.f;
#pragma unroll
        for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[32 * w + r][0]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            f[w] = __builtin_amdgcn_exp2f(ml[32 * w + r][0] - m);
            sum = fmaf(ml[32 * w + r][1], f[w], sum);
        }
        const uint32_t rt = ab_token(a, rr), head = kvh * group + rr - rt * group;
        const uint64_t to = ((uint64_t) tok_row + rt) * n_heads + head;
        const float inv = pieces > 1 ? 1.f : inverse(m, sum, ml[128 + r][0]);
#pragma unroll
        for (uint32_t k = 0; k < (uint32_t) DB; ++k) {
            const uint32_t quad = (tid & 7u) + 8u * k;
            if (4u * quad >= D) continue;
            float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float4_t x = ((const float4_t *) (tiles + w * S::BUF))[r * 8u * DB + (quad ^ (r & 7u))];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f[w], o[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] *= inv;
            if (pieces > 1) *(float4_t *) (a.rec_o + (rec + r) * D + 4u * quad) = o;
            else store(to, 4u * quad, o);
        }
        if (pieces > 1 && (tid & 7u) == 0u) *(float2_t *) (a.rec_ml + 2 * (rec + r)) = float2_t{m, sum};
        return;
    }
    together(std::false_type{});
    again_round = any_not_finite();
    if (again_round) together(std::true_type{});
    const float L = l_run + __shfl_xor(l_run, 32);
    uint32_t r = wave * 32u + n;  // the row again, computed anew: its registers are the key loop's until here
    asm volatile("" : "+v"(r));
    const uint32_t rr = tile * MOEARC_AB_ROWS + r;
    if (rr >= rows) return;
    const uint32_t rt = ab_token(a, rr), head = kvh * group + rr - rt * group;
    const uint64_t to = ((uint64_t) tok_row + rt) * n_heads + head;
    const float inv = pieces > 1 ? 1.f : inverse(m_run, L, sink2);
#pragma unroll
    for (int mb = 0; mb < DB; ++mb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t d = 32u * mb + 8u * j + 4u * h;
            if (d >= D) continue;
            const float4_t v = {O[mb][4 * j] * inv, O[mb][4 * j + 1] * inv, O[mb][4 * j + 2] * inv, O[mb][4 * j + 3] * inv};
            if (pieces > 1) *(float4_t *) (a.rec_o + (rec + r) * D + d) = v;
            else store(to, d, v);
        }
    if (pieces > 1 && h == 0) *(float2_t *) (a.rec_ml + 2 * (rec + r)) = float2_t{m_run, L};
}

// Joins the records of the tiles that were cut, in one pass over a row's pieces with the running maximum. A thread has
// four channels of a row; work-groups are (tile and KV head, 256 / (head_dim / 4) rows of it).
__device__ __forceinline__ void ab_merge_body(const AttnBatchArgs &a) {
    const uint32_t G = a.n_kv_heads, D = a.head_dim;
    const uint32_t at = (uint32_t) ((uint64_t) blockIdx.x * a.kv_magic >> a.kv_shift), kvh = blockIdx.x - at * G;
    const uint32_t b = a.n_slots > 1u ? ab_slot(a.merge_begin, at) : 0u;
    const AttnBatchSlot sl = a.slot[b];
    const uint32_t tile = at - sl.merge_begin, pieces = sl.pieces;
    const uint32_t rows = sl.n_new * a.group, tile_rows = sl.tile_rows;
    const uint32_t quads = D / 4u, r = blockIdx.y * (256u / quads) + threadIdx.x / quads, d = 4u * (threadIdx.x % quads);
    const uint32_t row = tile * tile_rows + r;
    if (threadIdx.x / quads >= 256u / quads || r >= tile_rows || row >= rows) return;
    const AbSpan span = ab_span(a, sl.n_new, sl.n_kv, tile, tile_rows);
    const uint32_t np = span.hi > span.lo ? (span.hi - span.lo + sl.piece - 1u) / sl.piece : 1u;
    const uint64_t rec0 = ((uint64_t) sl.rec_begin + tile * pieces * tile_rows) * G + kvh * tile_rows + r;
    const uint64_t step = (uint64_t) G * tile_rows;  // records from piece to piece
    const uint32_t tok = ab_token(a, row), hd = kvh * a.group + row - tok * a.group;
    const float sink2 = a.sinks ? ab_sink(a.sinks[hd]) : -INFINITY;
    float top = fmaxf(sink2, PF_M_INIT), total = __builtin_amdgcn_exp2f(sink2 - top + MOEARC_AB_LOG2_PSCALE);
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t k0 = 0; k0 < np; k0 += 8u) {  // eight records' loads at a time
        float2_t ml[8];
        float4_t x[8];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) {
            const uint64_t rec = rec0 + min(k0 + k, np - 1u) * step;
            ml[k] = *(const float2_t *) (a.rec_ml + 2 * rec);
            x[k] = *(const float4_t *) (a.rec_o + rec * D + d);
            if (k0 + k >= np) ml[k] = float2_t{PF_M_INIT, 0.f}, x[k] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        float m = top;
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) m = fmaxf(m, ml[k][0]);
        const float corr = __builtin_amdgcn_exp2f(top - m);
        top = m;
        total *= corr;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= corr;
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) {
            const float f = __builtin_amdgcn_exp2f(ml[k][0] - m);
            total = fmaf(ml[k][1], f, total);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[k][e], f, o[e]);
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const uint64_t to = (((uint64_t) sl.row0 + tok) * a.n_heads + hd) * D + d;
    if (a.out_f16) {
        const half2_t h0 = {(_Float16) (o[0] * inv), (_Float16) (o[1] * inv)}, h1 = {(_Float16) (o[2] * inv), (_Float16) (o[3] * inv)};
        *(u32x2_t *) ((_Float16 *) a.out + to) = u32x2_t{__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1)};
    } else {
        *(float4_t *) ((float *) a.out + to) = float4_t{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    }
}

}  // namespace

#define AB_KERNEL(DB, WAVES)                                                                                       \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES)))           \
    moearc_attn_batch_d##DB##_k(AttnBatchArgs a) {                                                                 \
        ab_body<DB, false>(a);                                                                                     \
    }                                                                                                              \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES)))           \
    moearc_attn_batch_precise_d##DB##_k(AttnBatchArgs a) {                                                         \
        ab_body<DB, true>(a);                                                                                      \
    }
AB_KERNEL(2, 3)
AB_KERNEL(4, 2)
AB_KERNEL(8, 1)
extern "C" __global__ void __launch_bounds__(256) moearc_attn_batch_merge_k(AttnBatchArgs a) { ab_merge_body(a); }
