// Attention of a ragged batch's new tokens over the paged f16 cache: sequences with any number of new
// tokens each (decode steps, drafts, prompt chunks), heads of up to 256 channels, any group and page size.
// Row (token i of n new ones, head) of a sequence with n_kv keys sits at p = n_kv - n + i and attends keys
// [max(0, p + 1 - n_swa), p] (n_swa 0: [0, p]) with the head's sink in the denominator; a row at p < 0 sees
// nothing and is zero.
//
// A work-group owns one KV head and a tile of 128 rows, a row being a (token, head of the KV head's group) pair, so
// K and V are read once for all of a tile's heads; its four waves take 32 rows each. Keys stream through LDS in
// 32-key tiles, four buffers, copies (LDS DMA, 16 bytes a lane) three tiles ahead, one barrier a tile. A tile whose
// keys are cut into pieces (few rows, many keys) leaves records that the merge kernel joins.
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
// A work-group that ends with a non-finite accumulator runs once more, with the tiles that cross a mask done key by key.
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

// LDS DMA of 16 bytes per lane of `mask` to LDS address lds + 16 * lane, from a lane's own address or from a
// wave-uniform one plus a lane's offset. Through asm: for the builtin the compiler, which cannot tell the buffer being
// read from the one being filled, would wait for the copy before every LDS read, and branch around it for the mask.
// m0 and exec are the compiler's: saved and restored; every lane is active where these are called.
__device__ __forceinline__ void ab_copy16(const uint8_t *p, uint32_t lds, uint64_t mask) {
    uint32_t m0_saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_mov_b64 exec, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t"
                 "s_mov_b64 exec, -1\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0_saved) : "v"(p), "s"(lds), "s"(mask) : "memory");
}
__device__ __forceinline__ void ab_copy16(const uint8_t *base, uint32_t off, uint32_t lds, uint64_t mask) {
    uint32_t m0_saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_mov_b64 exec, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
                 "s_mov_b64 exec, -1\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0_saved) : "v"(off), "s"(base), "s"(lds), "s"(mask) : "memory");
}

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

// Keys [lo, hi) that the rows of tile t of a slot see. No other's block-table entry is looked at.
struct AbSpan {
    uint32_t lo, hi;
};
__device__ __forceinline__ AbSpan ab_span(const AttnBatchArgs &a, uint32_t b, uint32_t t) {
    const uint32_t n = a.n_new[b];
    const int32_t shift = (int32_t) (a.n_kv[b] - n);  // a token's position less its index; below 0: the first see nothing
    const uint32_t tok0 = t * MOEARC_AB_ROWS / a.group, tok1 = min((t * MOEARC_AB_ROWS + MOEARC_AB_ROWS - 1u) / a.group, n - 1u);
    const int32_t last = shift + (int32_t) tok1, first = max(0, shift + (int32_t) tok0);
    AbSpan s;
    s.hi = last < 0 ? 0u : (uint32_t) last + 1u;
    s.lo = a.n_swa && (uint32_t) first + 1u > a.n_swa ? (uint32_t) first + 1u - a.n_swa : 0u;
    if (a.page_tokens % 8u == 0u) s.lo &= ~7u;  // in the same page
    return s;
}

template <int DB, bool PRECISE>
__device__ __forceinline__ void ab_body(const AttnBatchArgs &a) {
    using S = AbShape<DB>;
    constexpr int NBUF = 4;
    __shared__ __attribute__((aligned(1024))) uint8_t tiles[NBUF * S::BUF];
    __shared__ uint32_t table[MOEARC_AB_PT];  // places in the pools (page * page_tokens + slot) of eight keys each, or of each key
    __shared__ uint32_t again;

    const uint32_t tid = threadIdx.x, lane = tid & 63u, h = lane >> 5, n = lane & 31u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t G = a.n_kv_heads, D = a.head_dim, group = a.group;
    const uint32_t kvh = blockIdx.x % G, item = blockIdx.x / G;
    const uint32_t b = ab_slot(a.item_begin, item);
    const uint32_t nt = a.n_tiles[b], in_slot = item - a.item_begin[b];
    const uint32_t pieces = (a.item_begin[b + 1] - a.item_begin[b]) / nt;
    const uint32_t pc = in_slot / nt, tile = nt - 1u - in_slot % nt;  // the latest tile, which has the most keys, first
    const AbSpan span = ab_span(a, b, tile);
    const uint32_t lo = span.lo + pc * a.piece;  // with pages of eights a multiple of 8
    const uint32_t hi = pieces > 1 ? min(span.hi, lo + a.piece) : span.hi;
    if (pc && lo >= span.hi) return;  // an earlier tile's span has fewer pieces

    // ---- this lane's query row ------------------------------------------------------------------
    const uint32_t n_new = a.n_new[b], rows = n_new * group;
    const int32_t shift = (int32_t) (a.n_kv[b] - n_new);
    const uint32_t row = tile * MOEARC_AB_ROWS + wave * 32u + n;
    const bool row_ok = row < rows;
    const uint32_t tok = min(row, rows - 1u) / group, hd = kvh * group + min(row, rows - 1u) % group;
    const int32_t pos = shift + (int32_t) tok;
    // visible keys j: j - row_lo <= row_len as unsigned numbers (an empty row: at 2^31, which no key has)
    const uint32_t row_lo = pos < 0 ? 0x80000000u : a.n_swa && (uint32_t) pos + 1u > a.n_swa ? (uint32_t) pos + 1u - a.n_swa : 0u;
    const uint32_t row_len = pos < 0 ? 0u : (uint32_t) pos - row_lo;
    const uint64_t out_row = ((uint64_t) a.row0[b] + tok) * a.n_heads + hd;
    half8_t qop[2 * DB];
#pragma unroll
    for (int t = 0; t < 2 * DB; ++t) {
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (row_ok && 16u * t + 8u * h < D) v = *(const u32x4_t *) (a.q + out_row * D + 16u * t + 8u * h);
        qop[t] = __builtin_bit_cast(half8_t, v);
    }
    float c = a.scale_log2e;
    if (c < 0.f) {  // s * c = (-s) * (-c): then the row maximum of s * c is c times the maximum of s
        c = -c;
#pragma unroll
        for (int t = 0; t < 2 * DB; ++t) qop[t] = -qop[t];
    }
    if (c == 0.f) {  // every score 0, and masked ones still -inf: q = 0
        c = 1.f;
#pragma unroll
            for (int t = 0; t < 2 * DB; ++t) qop[t] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
    }
    // q has arrived: the compiler would wait for its loads in the key loop, and so for the copies issued after them
#pragma unroll
    for (int t = 0; t < 2 * DB; ++t) asm volatile("" : "+v"(qop[t]));
    // positions of the wave's first and last row: which tiles cross a mask
    const uint32_t wr0 = tile * MOEARC_AB_ROWS + wave * 32u;
    const int32_t w_first = shift + (int32_t) (min(wr0, rows - 1u) / group);
    const int32_t w_last = shift + (int32_t) (min(wr0 + 31u, rows - 1u) / group);
    const int32_t w_lo_last = a.n_swa ? max(0, w_last + 1 - (int32_t) a.n_swa) : 0;

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
    const bool eights = a.page_tokens % 8u == 0u;
    // Byte offsets from its first key's row in the pool of what this lane copies of a wave's eight keys, and whether there
    // is such a chunk in a head.
    uint32_t off_k[S::COPIES], off_v[S::COPIES];
    uint64_t has_k[S::COPIES], has_v[S::COPIES];
#pragma unroll
    for (uint32_t i = 0; i < S::COPIES; ++i) {
        const uint32_t key = ld_key + i * S::KEYS, ck = ld_slot ^ S::fk(8u * wave + key), cv = ld_slot ^ S::fv(8u * wave + key);
        off_k[i] = key * key_bytes + head_bytes + 16u * ck;
        off_v[i] = key * key_bytes + head_bytes + 16u * cv;
        has_k[i] = __builtin_amdgcn_ballot_w64(8u * ck < D);
        has_v[i] = __builtin_amdgcn_ballot_w64(8u * cv < D);
    }
    if (D < 32u * DB) {  // chunks behind the head's channels are never copied: zeros for the products
        for (uint32_t i = tid; i < NBUF * S::BUF / 16u; i += 256u) ((u32x4_t *) tiles)[i] = u32x4_t{0u, 0u, 0u, 0u};
    }

    float m_run, l_run;
    float16_t O[DB];
    const half2_t ones2 = {1, 1};
    const uint32_t *row_table = a.block_tables + a.seq[b] * a.bt_stride;

    auto all_keys = [&](auto by_key_c) {
        constexpr bool BY_KEY = decltype(by_key_c)::value;
        m_run = PF_M_INIT;
        l_run = 0.f;
#pragma unroll
        for (int mb = 0; mb < DB; ++mb)
#pragma unroll
            for (int i = 0; i < 16; ++i) O[mb][i] = 0.f;

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

        // S^T of the tile in buffer buf.
        auto scores = [&](uint32_t buf) {
            const uint8_t *const kt = tiles + buf * S::BUF;
            float16_t s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
            for (int t = 0; t < 2 * DB; ++t)
                s = pf_mfma(*(const half8_t *) (kt + (k_at ^ (uint32_t) t << 5)), qop[t], s);
            return s;
        };
        // The tile of keys j0 .. in buffer buf, s its scores; the next tile's scores, whose products run beside the
        // weights' arithmetic.
        auto compute = [&](float16_t s, uint32_t j0, uint32_t buf, uint32_t next_buf) -> float16_t {
            const uint8_t *const kt = tiles + buf * S::BUF;
            const bool masked = (int32_t) j0 + 31 > w_first || (int32_t) j0 < w_lo_last;
            if (masked) {
                const uint32_t off = j0 + 4u * h - row_lo;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (off + (uint32_t) (8 * (i >> 2) + (i & 3)) > row_len) s[i] = -INFINITY;
            }
            const float16_t next = scores(next_buf);
            half8_t phi[2], plo[2];
            float l = weights(s, MOEARC_AB_LOG2_PSCALE - m_run, l_run, phi, plo);
            if (__builtin_amdgcn_ballot_w64(l == INFINITY) != 0) {
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
                l = weights(s, MOEARC_AB_LOG2_PSCALE - m_run, l_run, phi, plo);
            }
            if constexpr (PRECISE) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2((half2_t){plo[q][i], plo[q][i + 1]}, ones2, l, false);
            }
            l_run = l;
            if (BY_KEY && masked) {  // weight and visibility from the lane that holds them
                for (uint32_t k = 0; k < 32u; ++k) {
                    const uint32_t i = 4u * (k >> 3) + (k & 3u);  // register of lane half (k >> 2) & 1
                    float w = 0.f;
#pragma unroll
                    for (uint32_t r = 0; r < 16u; ++r)
                        if (r == i) w = (float) phi[r >> 3][r & 7] + (PRECISE ? (float) plo[r >> 3][r & 7] : 0.f);
                    w = __shfl(w, (int) (n + 32u * ((k >> 2) & 1u)));
                    const bool sees = j0 + k - row_lo <= row_len;
#pragma unroll
                    for (int mb = 0; mb < DB; ++mb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const uint32_t ch = 32u * mb + 8u * (r >> 2) + 4u * h + (r & 3u);
                            const float v = (float) *(const _Float16 *) (kt + S::TILE + S::v_at(k, ch >> 3) + 2u * (ch & 7u));
                            if (sees) O[mb][r] = fmaf(w, v, O[mb][r]);
                        }
                }
                return next;
            }
#pragma unroll
            for (int mb = 0; mb < DB; ++mb)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint8_t *p = kt + v_at[mb] + q * 16 * S::ROW;
                    const short4v_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t *) p);
                    const short4v_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t *) (p + 8 * S::ROW));
                    typedef short short8v_t __attribute__((ext_vector_type(8)));
                    const short8v_t x = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
                    const half8_t va = __builtin_bit_cast(half8_t, x);
                    O[mb] = pf_mfma(va, phi[q], O[mb]);
                    if constexpr (PRECISE) O[mb] = pf_mfma(va, plo[q], O[mb]);
                }
            return next;
        };

        // Keys whose places fit `table` at a time; one step computes a 32-key tile.
        const uint32_t seg_keys = eights ? 8u * MOEARC_AB_PT : MOEARC_AB_PT;
        for (uint32_t seg = lo; seg < hi; seg += seg_keys) {
            const uint32_t seg_hi = min(hi, seg + seg_keys), last_key = seg_hi - 1u;
            const uint32_t n_places = eights ? (last_key - seg) / 8u + 1u : last_key - seg + 1u;
            __syncthreads();
            for (uint32_t i = tid; i < n_places; i += 256u) {
                const uint32_t key = seg + (eights ? 8u * i : i);
                const uint32_t page = (uint32_t) ((uint64_t) key * a.page_magic >> a.page_shift);
                uint32_t id = row_table[page];
                if (id >= a.n_pages) {  // reported; what is read instead lies in the pool
                    *(volatile uint32_t *) a.err = 1u;
                    id = 0u;
                }
                table[i] = id * a.page_tokens + (key - page * a.page_tokens);
            }
            __syncthreads();
            // A wave's copies of a tile: its eight keys of K and of V. With pages of eights these share a page, and their
            // base is wave-uniform. Keys behind the last are that one: their scores are masked, and no slot is read that the
            // cache has not written.
            auto copy_tile = [&](uint32_t j0, uint32_t buf) {
                const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + buf * S::BUF + 8u * wave * S::ROW), j = j0 + 8u * wave;
                if (eights && j + 7u <= last_key) {
                    const uint64_t at = (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) table[(j - seg) / 8u]) * key_bytes;
#pragma unroll
                    for (uint32_t i = 0; i < S::COPIES; ++i) {
                        ab_copy16((const uint8_t *) a.k_pages + at, off_k[i], dst + i * 1024u, has_k[i]);
                        ab_copy16((const uint8_t *) a.v_pages + at, off_v[i], dst + S::TILE + i * 1024u, has_v[i]);
                    }
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < S::COPIES; ++i) {
                        const uint32_t key = ld_key + i * S::KEYS, at_key = min(j + key, last_key) - seg;
                        const uint32_t place = eights ? table[at_key / 8u] + at_key % 8u : table[at_key];
                        const uint64_t at = (uint64_t) place * key_bytes;
                        const uint32_t less = key * key_bytes;
                        ab_copy16((const uint8_t *) a.k_pages + at + (off_k[i] - less), dst + i * 1024u, has_k[i]);
                        ab_copy16((const uint8_t *) a.v_pages + at + (off_v[i] - less), dst + S::TILE + i * 1024u, has_v[i]);
                    }
                }
            };
            // Step r: this wave's copies of tile r + 1 are done (those of r + 2, issued later, may be in flight), every
            // wave meets, so all copies of r + 1 are in and nobody reads tile r - 1's buffer, which r + 3 then takes.
            // Tiles behind the last are copied again, into buffers whose scores nobody uses, so the count is always the same.
            const uint32_t steps = (seg_hi - seg + 31u) / 32u;
            auto first_key = [&](uint32_t r) { return seg + 32u * min(r, steps - 1u); };
#pragma unroll
            for (uint32_t r = 0; r < NBUF - 1; ++r) copy_tile(first_key(r), r);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((NBUF - 2) * 2 * S::COPIES) : "memory");
            float16_t s = scores(0);
            for (uint32_t r = 0; r < steps; ++r) {
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((NBUF - 3) * 2 * S::COPIES) : "memory");
                copy_tile(first_key(r + NBUF - 1u), (r + NBUF - 1u) % NBUF);
                s = compute(s, first_key(r), r % NBUF, (r + 1u) % NBUF);
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");  // before the buffers are filled again, or released
        }

    };
    all_keys(std::false_type{});
    bool finite = true;
    if (row_ok) {
#pragma unroll
        for (int mb = 0; mb < DB; ++mb)
#pragma unroll
            for (int i = 0; i < 16; ++i) finite = finite && (__float_as_uint(O[mb][i]) & 0x7F800000u) != 0x7F800000u;
    }
    __syncthreads();
    if (tid == 0) again = 0u;
    __syncthreads();
    if (!finite) again = 1u;
    __syncthreads();
    if (again) all_keys(std::true_type{});

    const float L = l_run + __shfl_xor(l_run, 32);
    if (!row_ok) return;
    if (pieces > 1) {
        const uint64_t rec = ((uint64_t) (a.rec_begin[b] + tile * pieces + pc) * G + kvh) * MOEARC_AB_ROWS + wave * 32u + n;
        float *o = a.rec_o + rec * D;
#pragma unroll
        for (int mb = 0; mb < DB; ++mb)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t d = 32u * mb + 8u * j + 4u * h;
                if (d < D) *(float4_t *) (o + d) = float4_t{O[mb][4 * j], O[mb][4 * j + 1], O[mb][4 * j + 2], O[mb][4 * j + 3]};
            }
        if (h == 0) *(float2_t *) (a.rec_ml + 2 * rec) = float2_t{m_run, L};
        return;
    }
    const float sink2 = a.sinks ? a.sinks[hd] * MOEARC_LOG2E : -INFINITY;
    const float top = fmaxf(m_run, sink2);
    const float fm = __builtin_amdgcn_exp2f(m_run - top);
    const float total = L * fm + __builtin_amdgcn_exp2f(sink2 - top + MOEARC_AB_LOG2_PSCALE);
    const float inv = total == 0.f ? 0.f : fm / total;  // a row without keys and without a sink
#pragma unroll
    for (int mb = 0; mb < DB; ++mb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t d = 32u * mb + 8u * j + 4u * h;
            if (d >= D) continue;
            const float4_t v = {O[mb][4 * j] * inv, O[mb][4 * j + 1] * inv, O[mb][4 * j + 2] * inv, O[mb][4 * j + 3] * inv};
            if (a.out_f16) {
                const half2_t h0 = {(_Float16) v[0], (_Float16) v[1]}, h1 = {(_Float16) v[2], (_Float16) v[3]};
                *(u32x2_t *) ((_Float16 *) a.out + out_row * D + d) =
                    u32x2_t{__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1)};
            } else {
                *(float4_t *) ((float *) a.out + out_row * D + d) = v;
            }
        }
}

// Joins the records of the tiles that were cut: a work-group takes rows_per_block rows of one tile and KV head, a row
// its head_dim / 4 neighbouring lanes' worth of work, float4 each.
__device__ __forceinline__ void ab_merge_body(const AttnBatchArgs &a) {
    const uint32_t G = a.n_kv_heads, D = a.head_dim, kvh = blockIdx.x % G, at = blockIdx.x / G;
    const uint32_t b = ab_slot(a.merge_begin, at);
    const uint32_t nt = a.n_tiles[b], tile = at - a.merge_begin[b], pieces = (a.item_begin[b + 1] - a.item_begin[b]) / nt;
    const AbSpan span = ab_span(a, b, tile);
    const uint32_t np = span.hi > span.lo ? (span.hi - span.lo + a.piece - 1u) / a.piece : 1u;
    const uint32_t rows = min((uint32_t) MOEARC_AB_ROWS, a.n_new[b] * a.group - tile * MOEARC_AB_ROWS);
    const uint32_t quads = D / 4u;
    const uint64_t rec0 = ((uint64_t) (a.rec_begin[b] + tile * pieces) * G + kvh) * MOEARC_AB_ROWS;
    const uint64_t step = (uint64_t) G * MOEARC_AB_ROWS;  // records from piece to piece
    const uint32_t r_end = min(rows, (blockIdx.y + 1u) * a.rows_per_block);
    for (uint32_t i = threadIdx.x + blockIdx.y * a.rows_per_block * quads; i < r_end * quads; i += 256u) {
        const uint32_t r = i / quads, d = 4u * (i % quads);
        const uint32_t row = tile * MOEARC_AB_ROWS + r, tok = row / a.group, hd = kvh * a.group + row % a.group;
        const float sink2 = a.sinks ? a.sinks[hd] * MOEARC_LOG2E : -INFINITY;
        float top = fmaxf(sink2, PF_M_INIT);
        for (uint32_t k = 0; k < np; ++k) top = fmaxf(top, a.rec_ml[2 * (rec0 + k * step + r)]);
        float total = __builtin_amdgcn_exp2f(sink2 - top + MOEARC_AB_LOG2_PSCALE);
        float4_t o = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t k = 0; k < np; ++k) {
            const uint64_t rec = rec0 + k * step + r;
            const float2_t ml = *(const float2_t *) (a.rec_ml + 2 * rec);
            const float f = __builtin_amdgcn_exp2f(ml[0] - top);
            const float4_t x = *(const float4_t *) (a.rec_o + rec * D + d);
            total = fmaf(ml[1], f, total);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const uint64_t to = (((uint64_t) a.row0[b] + tok) * a.n_heads + hd) * D + d;
        if (a.out_f16) {
            const half2_t h0 = {(_Float16) (o[0] * inv), (_Float16) (o[1] * inv)}, h1 = {(_Float16) (o[2] * inv), (_Float16) (o[3] * inv)};
            *(u32x2_t *) ((_Float16 *) a.out + to) = u32x2_t{__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1)};
        } else {
            *(float4_t *) ((float *) a.out + to) = float4_t{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        }
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
