// Paged decode attention split over the keys (gfx950): caches in bf16 or microscaled elements (mx_format.h), and groups of
// sequences that share a prefix.
//
// For a row (query token, query head) with keys partitioned into pieces p, each piece gives
//     m_p = max_j s_j,  l_p = sum_j 2^(s_j - m_p),  O_p = sum_j 2^(s_j - m_p) v_j        (s in units of log2)
// and the row's output is  sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p,  m = max_p m_p.  A prefix shared by a group is a piece like
// any other, computed for the rows of ALL the group's sequences at once: its keys are read once per row tile instead of
// once per sequence, and the matrix instructions get full tiles where a sequence alone has a few rows.
//
// Work list: "virtual sequences" -- the groups (rows: all tokens of the group's sequences; keys: the prefix, through the first
// sequence's block table) and then the sequences (keys: the context behind the prefix, then the fresh rows).  An item
// is (virtual sequence, KV head or heads, row tile), a unit one key tile of it; items are dealt to the workgroups in
// contiguous ranges of equal cost, cut where a range ends.  Every workgroup works the list out for itself from the lengths on the device (no
// host read, safe in a captured graph with later lengths); the last launch merges the pieces.
//
// Two kinds of items, chosen by the rows, each with a launch of its own (they want different register budgets):
//   narrow (single tokens, small blocks): bound by memory.  32 rows; four waves, each with a KV head of its own where there are
//     four (a token's codes and scales of neighbouring heads lie in the same memory lines: the waves of a workgroup should want them
//     at the same time), with every second or fourth tile of a head otherwise, whose softmax states are then merged in LDS.
//     A wave moves its 32-key tiles into LDS of its own: no barrier in the loop, the next tiles' loads issued before the arithmetic
//     (how far they stay in flight over it: kDepth).
//     5 single tokens of 32 / 32 heads over 20000 to 60000 E2M1 keys: 275 us, 3.0 TB/s (425 us with a workgroup's waves on four tiles of one
//     head: a head's 4 scale bytes and 64 codes are a part of a memory line each).
//   wide: bound by the matrix instructions and the exponentials.  256 rows, 32 for each of eight waves, over 64-key tiles shared by the
//     waves; in each wave the products of one tile's scores run beside the exponentials of the tile before.
//     128 sequences of 32 tokens, 28 / 4 heads, over 2048 to 8192 E4M3 keys: 420 to 455 us, 680 to 735 TFLOP/s of the rows' own products (224 of a tile's
//     256 rows).  Two row blocks per wave (half the LDS reads) do not fit the registers; one launch for both kinds, sharing the workgroups out,
//     gained 7 us where a prefix of 4096 serves 64 single tokens and lost 8 to 17 us elsewhere.
// At head_dim 128 both kinds take all 256 registers and spill some 60 to 85: the wide ones around an item (bf16 four in a tile's step as well), the
// narrow ones in the loop.
// Microscaled codes are widened on the way from registers to LDS, once per tile, with their block's scale applied by the same
// instruction: from there on the arithmetic is the bf16 cache's.
#include "attn_tile.h"
#include "mx_format.h"

namespace dfx {
namespace {

constexpr int kNarrowRows = 32, kWideRows = 256;
constexpr int kNarrowKeys = 32, kWideKeys = 64;
// Rows of a virtual sequence up to which its items are narrow.  Each tile of 32 rows reads the keys again, a wide tile costs the same whatever its rows.
// (Narrow against wide, E4M3, 4 KV heads, us: 32 rows over 4096 keys, 64 sequences: 110, 123; 64 rows: 143, 137; 96 rows: 219, 141, a bf16 cache 356,
// 176; 96 rows, 4 sequences: 47, 38; 64 rows over 700 keys, 128 sequences: 79, 87; 84 rows over 16 to 700 keys beside 4 prefixes of 8192: 320, 337:
// by the rows alone the last two take the slower side, by 5 to 10 %, for the 4 to 50 % of the others.)
constexpr int kNarrowMost = 32;
// Beside its units (cost 1 each) an item costs its start and end: queries, first tiles, the merge of the waves, the rows written.
// (Narrow: of the tiles that the waves of a head take side by side; a unit is one such tile.)
constexpr int kNarrowTail = 2, kWideTail = 3;
// Least cost per workgroup.  Shorter pieces take the merge longer than they save: 64 single tokens with a prefix of 4096 take 70, 66, 68 us with 2, 4, 6 for
// the wide, 8 tokens over 100 to 1000 keys 24.5, 25.7, 27.1 us with 2, 3, 4 for the narrow ones.
constexpr int kNarrowLeast = 2, kWideLeast = 4;

enum { kBf16 = 0, kMx8 = 1, kMx4 = 2 };

struct SplitArgs {
    const uint16_t* q;
    const uint16_t* k_new;
    const uint16_t* v_new;
    uint16_t* out;
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
    const int32_t* block_tables;
    const int32_t* context_lens;
    const int32_t* cu_q;
    const int32_t* cu_new;
    const int32_t* group_cu;
    const int32_t* group_len;
    uint8_t* workspace;
    int64_t q_st, q_sh, kn_st, kn_sh, vn_st, vn_sh, o_st, o_sh;
    uint32_t c_sp, c_st, c_sh;  // cache strides in bytes: page, token, head
    int64_t bt_stride;
    int64_t rec_off, comb_off, slot_off, ml_off;  // workspace
    int64_t n_slots[2], first_slot[2];            // piece slots (32 rows each) of the narrow and the wide items
    int n_pages, n_q, n_new;
    int n_seqs, n_groups, h_kv, group_heads;
    int page_size, page_shift, max_pages, dbs, block_causal, use_wide;
    int n_wg[2];  // working workgroups of the narrow and the wide launch
    int heads_shift;  // a narrow workgroup's KV heads: 1, 2 or 4 = 1 << heads_shift
    float c;  // scale * log2(e)
};

struct Header {    // one per kind
    int64_t total;   // cost of all items
    int32_t n_wg;    // workgroups that have work
    int32_t n_comb;  // row blocks of the merge (narrow launch)
};
struct Rec {         // a virtual sequence, for the merge
    int64_t cost;    // of the items of its kind before it
    int32_t blocks;  // row-block slots of the items of its kind before it
    int32_t tok0, rows, tiles, row_tiles;
    int32_t group;   // the group whose item covers a part of its keys, or -1
    int32_t narrow, has_keys;
};

struct Seq {
    int tok0, rows;          // first query token; rows of one KV head (tokens * heads of the group)
    int key0, key1;          // cached keys [key0, key1)
    int new0, n_new;         // fresh rows
    int table;               // block-table row
    int prefix;              // keys of this sequence's context that its group's item covers
    int seq0, seq1;          // sequences of the item
    int tiles, ctx_tiles, row_tiles;
    bool narrow;
    int group;               // its group, or -1
};
template <bool WIDE>
struct Kind {
    static constexpr int kWaves = WIDE ? 8 : 4, kThreads = kWaves * 64;
};
// What differs between the kinds and depends on the heads: the waves of a narrow workgroup that share a head take `side` tiles side by
// side.
struct Costs {
    int tail, least;    // in tiles
    int heads, blocks;  // KV heads of an item, slots of its pieces
    DFX_D Costs(const SplitArgs& a, bool narrow) {
        const int side = narrow ? Kind<false>::kWaves >> a.heads_shift : 1;
        tail = narrow ? kNarrowTail * side : kWideTail;
        least = narrow ? kNarrowLeast * side : kWideLeast;
        heads = narrow ? 1 << a.heads_shift : 1;
        blocks = narrow ? heads : kWideRows / 32;
    }
};
// An item of `tiles` units: unit u starts at cost u, the tail's cost lies behind the last.
DFX_D int item_cost(const Costs& k, int tiles) { return tiles > 0 ? tiles + k.tail : 0; }

DFX_D int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// The group of sequence s, -1 if it is in none.
DFX_D int group_of(const SplitArgs& a, int s) {
    int lo = 0, hi = a.n_groups;
    if (hi == 0 || s < a.group_cu[0] || s >= a.group_cu[hi]) return -1;
    while (hi - lo > 1) {  // the last group that starts at or before s
        const int mid = (lo + hi) >> 1;
        if (a.group_cu[mid] <= s) lo = mid;
        else hi = mid;
    }
    return lo;
}

DFX_D Seq seq_of(const SplitArgs& a, int v) {
    Seq q;
    const int64_t capacity = static_cast<int64_t>(a.max_pages) * a.page_size;
    // (keys are numbered in 32 bits, those of the tiles looked up ahead, up to 832 behind the last key, included)
    const int cap = static_cast<int>(capacity > INT32_MAX - 1024 ? INT32_MAX - 1024 : capacity);
    q.new0 = q.n_new = 0;
    q.group = -1;
    if (v < a.n_groups) {
        q.seq0 = clampi(a.group_cu[v], 0, a.n_seqs);
        q.seq1 = clampi(a.group_cu[v + 1], q.seq0, a.n_seqs);
        q.key0 = 0;
        q.key1 = q.prefix = clampi(a.group_len[v], 0, cap);
    } else {
        q.seq0 = v - a.n_groups;
        q.seq1 = q.seq0 + 1;
        q.key1 = clampi(a.context_lens ? a.context_lens[q.seq0] : 0, 0, cap);
        q.group = group_of(a, q.seq0);
        q.key0 = q.prefix = q.group < 0 ? 0 : clampi(a.group_len[q.group], 0, q.key1);
        q.new0 = clampi(a.cu_new[q.seq0], 0, a.n_new);
        q.n_new = clampi(a.cu_new[q.seq1], q.new0, a.n_new) - q.new0;
    }
    q.table = q.seq0;
    q.tok0 = clampi(a.cu_q[q.seq0], 0, a.n_q);
    q.rows = (clampi(a.cu_q[q.seq1], q.tok0, a.n_q) - q.tok0) * a.group_heads;
    q.narrow = !a.use_wide || q.rows <= kNarrowMost;
    const int kt = q.narrow ? kNarrowKeys : kWideKeys, rt = q.narrow ? kNarrowRows : kWideRows;
    q.row_tiles = (q.rows + rt - 1) / rt;
    q.ctx_tiles = (q.key1 - q.key0 + kt - 1) / kt;
    q.tiles = q.rows > 0 ? q.ctx_tiles + (q.n_new + kt - 1) / kt : 0;
    return q;
}

// Workgroup ranges: workgroup w owns the units that start at a cost in [floor(w U / W), floor((w + 1) U / W)); so the owner of
// cost x is floor(((x + 1) W - 1) / U).  (A quotient in fp64, put right: a 64-bit integer division is a hundred instructions.)
DFX_D int64_t range_start(int w, int64_t total, int n_wg) { return w * total / n_wg; }
DFX_D int owner_of(int64_t cost, int64_t total, int n_wg) {
    const int64_t x = (cost + 1) * n_wg - 1;
    int64_t q = static_cast<int64_t>(static_cast<double>(x) / static_cast<double>(total));
    if (q * total > x) --q;
    else if ((q + 1) * total <= x) ++q;
    return static_cast<int>(q);
}

// ---- one wave's arithmetic ---------------------------------------------------------------------
// NB blocks of 32 rows: lane (col, half) holds, of row col of each, the scores of keys 8 g + 4 half + (0..3) and the outputs
// of elements d with the same pattern (S^T = K Q^T, O^T += V^T P^T: the probabilities leave the softmax in the layout the
// second product's operand wants).
template <int HD, int NB>
struct Wave {
    using L = TileLayout<HD>;
    static constexpr int NSLAB = HD / 16, NDB = HD / 32;
    f32x16 o[NDB][NB];
    bf16x8 q[NB][NSLAB];
    float m[NB], l[NB];
    int lane, col, half;
    uint32_t k_lane, v_lane;

    DFX_D explicit Wave(int lane_) : lane(lane_), col(lane_ & 31), half(lane_ >> 5) {
        k_lane = col * L::ROWB + ((half ^ L::swizzle(col)) * 16);
        const int g16 = lane >> 4, sl16 = lane & 15;
        const int lrow = (g16 >> 1) * 4 + (sl16 >> 2);
        const int c = (g16 & 1) * 2 + ((sl16 & 3) >> 1);
        v_lane = lrow * L::ROWB + ((c ^ L::swizzle(lrow)) * 16) + (sl16 & 1) * 8;
    }

    DFX_D void reset() {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b] = -INFINITY;
            l[b] = 0.0f;
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][b][i] = 0.0f;
        }
    }

    DFX_D void load_q(int b, const uint16_t* row) {  // nullptr: a lane without a row
#pragma unroll
        for (int s = 0; s < NSLAB; ++s) {
            u32x4 w = {0, 0, 0, 0};
            if (row != nullptr) w = *reinterpret_cast<const u32x4*>(row + s * 16 + half * 8);
            q[b][s] = __builtin_bit_cast(bf16x8, w);
        }
    }

    // The lane's value and the other half's (lane ^ 32), in either order.
    DFX_D static void both_halves(float v, float& x, float& y) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t r0 = r[0], r1 = r[1];  // (a bit_cast of the element itself reads element 0 for both)
        x = __builtin_bit_cast(float, r0);
        y = __builtin_bit_cast(float, r1);
    }
    DFX_D static float half_max(float v) {
        float x, y;
        both_halves(v, x, y);
        return fmaxf(x, y);
    }
    DFX_D static float half_sum(float v) {
        float x, y;
        both_halves(v, x, y);
        return x + y;
    }

    // Operands: 32 keys of one 16-wide slab of d; 16 keys (slab x of 32-key block t) of one 32-wide block of d, transposed.
    DFX_D bf16x8 read_k(uint32_t kt, int t, int sl) const {
        typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
        return *(const lds_bf16x8*)static_cast<uintptr_t>(((kt + k_lane) ^ (sl * 32)) + t * 32 * L::ROWB);
    }
    DFX_D bf16x8 read_v(uint32_t vt, int t, int x, int d) const {
        typedef short short4v __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) short4v lds_short4v;
        short4v r[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            r[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)static_cast<uintptr_t>(
                ((vt + v_lane) ^ (((d * 4) ^ L::swizzle(i * 8)) * 16)) + (t * 32 + x * 16 + i * 8) * L::ROWB));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
    template <int NT>
    static DFX_D void clear(f32x16 (&s)[NT][NB]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][b][i] = 0.0f;
    }
    template <int NT>
    DFX_D void scores(uint32_t kt, f32x16 (&s)[NT][NB]) const {
        constexpr int kAhead = 2;
        clear(s);
        bf16x8 k[kAhead + 1][NT];
#pragma unroll
        for (int sl = 0; sl < NSLAB + kAhead; ++sl) {
            if (sl < NSLAB) {
#pragma unroll
                for (int t = 0; t < NT; ++t) k[sl % (kAhead + 1)][t] = read_k(kt, t, sl);
            }
            if (sl >= kAhead) {
                const int c = sl - kAhead;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int b = 0; b < NB; ++b) s[t][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[c % (kAhead + 1)][t], q[b][c], s[t][b], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);  // (all operands first would not fit the registers)
            }
        }
    }

    template <int NT>
    DFX_D void hide(f32x16 (&s)[NT][NB], int b, uint64_t seen) const {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t bits = static_cast<uint32_t>(seen >> (32 * t)) >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!(bits & (1u << (8 * (i >> 2) + (i & 3))))) s[t][b][i] = -INFINITY;
        }
    }

    template <int NT>
    DFX_D float top_of(const f32x16 (&s)[NT][NB], int b) const {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][b][i]);
        return top;
    }

    // The running maximum moves only where a tile's is more than 2^8 above it (or there is none yet): the
    // weights then stay below 2^8, far inside bf16 and fp32, and the accumulators are rarely rescaled.
    DFX_D void raise(int b, float top) {
        if (__builtin_amdgcn_ballot_w64(top > m[b] + 8.0f)) {
            const float next = fmaxf(m[b], top);
            const float alpha = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[b] - next);
            m[b] = next;
            l[b] *= alpha;
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][b][i] *= alpha;
        }
    }

    DFX_D float base_of(int b) const { return m[b] == -INFINITY ? 0.0f : m[b]; }
    // Weights of 16 keys (score registers 8 x .. 8 x + 7), rounded to bf16 for the second product (its matrix instruction takes two bf16 operands,
    // and V has no more; half a step, 2^-8 of a weight, as the rounded output's own); returns the sum of the unrounded ones.
    static DFX_D float weights8(const f32x16& s, int x, float c, float base, bf16x8& p) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * x + i], c, -base));
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{e[2 * i], e[2 * i + 1]}, bf16x2));
        p = __builtin_bit_cast(bf16x8, w);
        return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    }
    template <int NT>
    DFX_D void weights(const f32x16 (&s)[NT][NB], float c, bf16x8 (&p)[NB][NT][2]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float base = base_of(b);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < 2; ++x) l[b] += weights8(s[t][b], x, c, base, p[b][t][x]);
        }
    }

    template <int NT>
    DFX_D void accumulate(uint32_t vt, const bf16x8 (&p)[NB][NT][2]) {
        constexpr int kSteps = 2 * NT * NDB, kAhead = 3;
        bf16x8 v[kAhead + 1];
#pragma unroll
        for (int st = 0; st < kSteps + kAhead; ++st) {
            if (st < kSteps) v[st % (kAhead + 1)] = read_v(vt, st / (2 * NDB), (st / NDB) & 1, st % NDB);
            if (st >= kAhead) {
                const int c = st - kAhead, t = c / (2 * NDB), x = (c / NDB) & 1, d = c % NDB;
#pragma unroll
                for (int b = 0; b < NB; ++b) o[d][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[c % (kAhead + 1)], p[b][t][x], o[d][b], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // The two halves of a wide tile's step, with the vector work of one tile between the matrix instructions of another and
    // the LDS operands requested some instructions ahead: an operand takes longer to arrive than a matrix instruction to run.
    // The scheduling barriers keep the source's order: left to itself the compiler puts the matrix instructions in a row (a wave waits at
    // the second until the first is through the pipeline), or all loads first, which does not fit the registers.
    static constexpr int kAheadK = 1;  // slabs
    static constexpr int kAheadV = 3;  // 16 keys x 32 elements each
    //   weights of s, scores of the next tile
    DFX_D void weights_and_scores(const f32x16 (&s)[2][NB], float c, bf16x8 (&p)[NB][2][2], uint32_t kt, f32x16 (&next)[2][NB]) {
        static_assert(NB == 1, "the weights of a slab's step are those of one row block");
        constexpr int kEach = 32 / NSLAB;  // weights per step
        clear(next);
        const float base = base_of(0);
        float sum = 0.0f;
        uint32_t w[2][8];  // pairs of weights
        bf16x8 k[kAheadK + 1][2];
#pragma unroll
        for (int sl = 0; sl < kAheadK; ++sl) {
            k[sl][0] = read_k(kt, 0, sl);
            k[sl][1] = read_k(kt, 1, sl);
        }
#pragma unroll
        for (int sl = 0; sl < NSLAB; ++sl) {
            if (sl + kAheadK < NSLAB) {
                k[(sl + kAheadK) % (kAheadK + 1)][0] = read_k(kt, 0, sl + kAheadK);
                k[(sl + kAheadK) % (kAheadK + 1)][1] = read_k(kt, 1, sl + kAheadK);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int j = 0; j < kEach / 2; j += 2) {
                    const int e = sl * kEach + i * (kEach / 2) + j, t = e >> 4;
                    const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][0][e & 15], c, -base));
                    const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][0][(e & 15) + 1], c, -base));
                    sum += w0 + w1;
                    w[t][(e & 15) >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{w0, w1}, bf16x2));
                    // (wanted here: otherwise they are all made behind the last matrix instruction)
                    asm volatile("" : "+v"(w[t][(e & 15) >> 1]), "+v"(sum));
                }
                next[i][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[sl % (kAheadK + 1)][i], q[0][sl], next[i][0], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l[0] += sum;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                p[0][t][x] = __builtin_bit_cast(bf16x8, u32x4{w[t][4 * x], w[t][4 * x + 1], w[t][4 * x + 2], w[t][4 * x + 3]});
    }
    //   outputs of a tile and the largest of the next tile's scores (this half's, unscaled)
    DFX_D void accumulate_and_top(uint32_t vt, const bf16x8 (&p)[NB][2][2], const f32x16 (&next)[2][NB], float (&top)[NB]) {
        bf16x8 v[kAheadV + 1];
        constexpr int kSteps = 4 * NDB;
        constexpr int kEach = 32 / kSteps;  // scores per step
        top[0] = -INFINITY;
#pragma unroll
        for (int i = 0; i < kAheadV; ++i) v[i] = read_v(vt, i / (2 * NDB), (i / NDB) & 1, i % NDB);
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            const int t = st / (2 * NDB), x = (st / NDB) & 1, d = st % NDB, n = st + kAheadV;
            if (n < kSteps) v[n % (kAheadV + 1)] = read_v(vt, n / (2 * NDB), (n / NDB) & 1, n % NDB);
            o[d][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[st % (kAheadV + 1)], p[0][t][x], o[d][0], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < kEach; ++i) top[0] = fmaxf(top[0], next[(st * kEach + i) >> 4][0][(st * kEach + i) & 15]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

DFX_D void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- a workgroup's items -----------------------------------------------------------------------
template <int HD, int KV, bool WIDE>
struct Split {
    using L = TileLayout<HD>;
    static constexpr int NB = 1;  // row blocks of a wave
    static constexpr int kWgWaves = Kind<WIDE>::kWaves, kWgThreads = Kind<WIDE>::kThreads;
    using W = Wave<HD, NB>;
    static constexpr int NDB = HD / 32;
    static constexpr int kRowBytes = KV == kBf16 ? HD * 2 : KV == kMx8 ? HD : HD / 2;  // codes of a head row
    static constexpr int kChunks = kRowBytes / 16;                                     // 16-byte chunks of them
    static constexpr int kNewChunks = HD / 8;                                          // of a fresh (bf16) row
    static constexpr int KT = WIDE ? kWideKeys : kNarrowKeys;
    static constexpr int ROWS = WIDE ? kWideKeys / kWgWaves : kNarrowKeys;             // rows of a tile that one wave moves
    static constexpr int kMat = KT * L::ROWB;                                          // K or V of a tile in LDS
    static constexpr int kLds = WIDE ? 6 * kMat : kWgWaves * 2 * kMat;                 // three buffers each; a tile per wave
    static constexpr int kAccBytes = 32 * HD * 4;
    static constexpr int kPer = 64 / kChunks;                                          // rows per load of the wave
    static constexpr int kLoads = ROWS > kPer ? ROWS / kPer : 1;                       // (one that some lanes only repeat, where ROWS < kPer)
    // Tiles in flight per wave of a narrow item, as far as the source goes: the eight waves of a compute unit should have some 100 KB on the way; a
    // bf16 tile is 16 KB.  Compiled for head_dim 128, E4M3 reloads spilled registers right behind a tile's loads, which waits for them all (no tile
    // stays in flight over the arithmetic), E2M1 waits for all loads in the first of its three steps only, bf16 reloads in front of its loads.
    static constexpr int kDepth = KV == kBf16 ? 1 : KV == kMx8 ? 2 : 3;
    static constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << 32) - 1;

    const SplitArgs& a;
    uint8_t* lds;
    float* ml;  // [4 waves][m, l][32]
    int tid, wave, lane;
    W w;
    // the item
    Seq sq;
    int kvh, row_tile;
    int lim_ctx[NB], lim_new[NB];  // this lane's rows see cached keys below lim_ctx and fresh rows below lim_new
    int key_end, new_end;          // cached keys and fresh rows from here on are zeros in LDS (see another_pass())
    uint64_t lane_off;             // of the KV head and of this lane's chunk, in a cache row
    uint32_t my_offset;            // stage_offset()
    const int32_t* table;          // the item's block-table row

    DFX_D Split(const SplitArgs& args, uint8_t* smem, float* ml_, int tid_)
        : a(args), lds(smem), ml(ml_), tid(tid_), wave(uniform(tid_ >> 6)), lane(tid_ & 63), w(tid_ & 63) {
        my_offset = stage_offset(lane, WIDE ? wave * ROWS : 0);
    }

    // Key `lane` of tile t: look_up() loads its page's table entry, row_of() -- a tile later, so that nothing waits for the load --
    // makes it the byte offset of the key's cache row (token) and tells which keys have none: fresh tiles, keys behind the last,
    // skipped pages (offset 0: the cache's first row).
    struct Key {
        int page, off;
        bool ok;
    };
    DFX_D Key look_up(int t) const {
        const int pos = sq.key0 + t * KT + lane;
        const int p = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page_size;
        Key k;
        k.ok = t < sq.ctx_tiles && lane < KT && pos < key_end && p < a.max_pages;
        k.off = pos - p * a.page_size;
        k.page = table[static_cast<uint32_t>(min(p, a.max_pages - 1))];
        return k;
    }
    DFX_D int64_t row_of(const Key& k, uint64_t& valid) const {
        const bool ok = k.ok && k.page >= 0 && k.page < a.n_pages;
        valid = __builtin_amdgcn_ballot_w64(ok);
        const uint32_t page = ok ? k.page : 0, off = ok ? k.off : 0;
        return static_cast<int64_t>(static_cast<uint64_t>(page) * a.c_sp + static_cast<uint64_t>(off) * a.c_st);
    }

    // The wave's share of a K or V tile on its way: loads i, rows r0 + stage_row(i), chunk lane % kChunks.
    struct Stage {
        u32x4 w[kLoads];
        uint8_t s[kLoads];
    };
    static DFX_D uint32_t address(const uint8_t* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)); }
    // Which of a load's rows a lane takes.  A chunk of codes becomes 2 or 4 chunks in LDS, which leave one per lane at a time: 16 lanes
    // should then write all 16 chunk positions of a 256-byte LDS line, i.e. lie on rows whose swizzles (TileLayout) differ where their
    // chunk indices agree, in the lowest bits -- that is row bits 2 and 3.
    static DFX_D int lane_row(int j) {
        if constexpr (KV == kBf16) return j;
        if constexpr (HD == 128 && KV == kMx8) return ((j & 1) << 2) | (j >> 1);                                   // of 8
        if constexpr (HD == 128 && KV == kMx4) return ((j & 3) << 2) | (j >> 2);                                   // of 16
        if constexpr (HD == 64 && KV == kMx8) return (j & 9) | ((j & 2) << 1) | ((j & 4) >> 1);                    // of 16
        return (j & 17) | ((j & 2) << 1) | ((j & 4) << 1) | ((j & 8) >> 2);                                        // of 32
    }
    DFX_D int stage_row(int i) const { return i * kPer + lane_row(lane / kChunks); }
    static DFX_D int64_t shuffle64(int64_t x, int from) {
        const int lo = __builtin_amdgcn_ds_bpermute(from * 4, static_cast<int>(x));
        const int hi = __builtin_amdgcn_ds_bpermute(from * 4, static_cast<int>(x >> 32));
        return static_cast<int64_t>(static_cast<uint32_t>(lo)) | (static_cast<int64_t>(hi) << 32);
    }
    // Issues the loads; `row` is row_of() the tile's keys.  No branch on the rows -- keys without a cache row load the cache's first
    // row and are zeroed in commit() -- so that the compiler can count the loads in flight.
    struct Place {
        uint64_t off[kLoads];
    };
    DFX_D Place place_of(int64_t row, int r0) const {
        Place p;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) p.off[i] = static_cast<uint64_t>(shuffle64(row, r0 + min(stage_row(i), ROWS - 1))) + lane_off;
        return p;
    }
    DFX_D void issue(Stage& st, const uint8_t* codes, const uint8_t* scales, const Place& p) const {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            st.w[i] = *reinterpret_cast<const u32x4*>(codes + p.off[i]);
            if constexpr (KV != kBf16) st.s[i] = scales[p.off[i] >> (KV == kMx8 ? 5 : 4)];
        }
    }
    // Byte offset in a tile in LDS of the first chunk that this lane writes of its load 0.  The chunks of a row and the rows of the other loads
    // differ from it in bits that no carry reaches, so that the swizzle's XOR can be applied to the finished address (TileMath).
    static constexpr int kWiden = KV == kBf16 ? 1 : KV == kMx8 ? 2 : 4;  // chunks in LDS per chunk of codes
    static DFX_D uint32_t stage_offset(int lane, int r0) {
        return L::chunk_offset(r0 + lane_row(lane / kChunks), lane % kChunks * kWiden);
    }
    // Registers -> LDS, widened.  valid: which keys of the tile have a cache row.
    DFX_D void commit(Stage& st, uint8_t* to, int r0, uint64_t valid) const {
        if (valid != kAll) {
            asm volatile("");  // (a branch of the wave: as selects the zeroing would cost every tile)
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (!((valid >> ((r0 + stage_row(i)) & 63)) & 1)) {
                    st.w[i] = u32x4{0, 0, 0, 0};
                    st.s[i] = 0;
                }
        }
        if (ROWS < kPer && stage_row(0) >= ROWS) return;
        typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
        const uint32_t at = address(to) + my_offset;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const float s = mx_scale_operand(st.s[i]);
#pragma unroll
            for (int x = 0; x < kWiden; ++x) {
                u32x4 y;
                if constexpr (KV == kBf16) y = st.w[i];
                else if constexpr (KV == kMx8) y = mx_widen8_e4m3(u32x2{st.w[i][2 * x], st.w[i][2 * x + 1]}, s);
                else y = mx_widen8_e2m1(st.w[i][x], s);
                *(lds_u32x4*)static_cast<uintptr_t>((at ^ ((x ^ L::swizzle(i * kPer)) * 16)) + i * kPer * L::ROWB) = y;
            }
        }
    }
    // Fresh rows (bf16 operands) of fresh tile t: straight to LDS, one after the other (a branch and a wait each), there are few of them.
    DFX_D void fresh_rows(const uint16_t* from, int64_t st, int64_t sh, int t, uint8_t* to, int r0) const {
        constexpr int kStep = 64 / kNewChunks;
#pragma unroll
        for (int i = 0; i < ROWS / kStep; ++i) {
            const int r = r0 + i * kStep + lane / kNewChunks, ch = lane % kNewChunks, j = t * KT + r;
            u32x4 x = {0, 0, 0, 0};
            if (j < new_end) x = *reinterpret_cast<const u32x4*>(from + (sq.new0 + static_cast<int64_t>(j)) * st + kvh * sh + ch * 8);
            *reinterpret_cast<u32x4*>(to + L::chunk_offset(r, ch)) = x;
        }
    }
    static DFX_D uint64_t below(int n) { return n <= 0 ? 0 : (n >= 64 ? ~0ull : (1ull << n) - 1); }

    // Scores of the keys that a row does not see: of context tile t, of fresh tile t (counted from the first fresh one).
    template <int NT>
    DFX_D void mask_context(f32x16 (&s)[NT][NB], int t, uint64_t valid) const {
        const int visible = lim_ctx[0] - (sq.key0 + t * KT);
        if (valid == kAll && __builtin_amdgcn_ballot_w64(visible < KT) == 0) return;
        w.hide(s, 0, below(visible) & valid);
    }
    template <int NT>
    DFX_D void mask_fresh(f32x16 (&s)[NT][NB], int t) const {
        const int visible = lim_new[0] - t * KT;
        if (__builtin_amdgcn_ballot_w64(visible < KT) == 0) return;
        w.hide(s, 0, below(visible));
    }
    // All of a tile's arithmetic.
    template <typename Mask>
    DFX_D void whole_tile(const uint8_t* kt, const uint8_t* vt, const Mask& mask) {
        constexpr int NT = KT / 32;
        f32x16 s[NT][NB];
        bf16x8 p[NB][NT][2];
        w.scores(address(kt), s);
        mask(s);
        w.raise(0, W::half_max(w.top_of(s, 0)) * a.c);
        w.weights(s, a.c, p);
        w.accumulate(address(vt), p);
    }

    // (one block of rows after the other, not a loop over them: a loop that holds another is unrolled too late for the compiler to
    // keep the state it indexes in registers)
    DFX_D void start_rows(int b, int rows_from, bool uneven) {
        const int row = rows_from + b * 32 + w.col;
        const bool live = row < sq.rows;
        const int t = live ? row / a.group_heads : 0, g = live ? row - t * a.group_heads : 0;
        const int64_t tok = sq.tok0 + t;
        w.load_q(b, live ? a.q + tok * a.q_st + (static_cast<int64_t>(kvh) * a.group_heads + g) * a.q_sh : nullptr);
        int ctx = live ? sq.key1 : INT32_MAX;
        if (uneven && live) {  // the row's sequence may end inside the prefix, or before it
            int lo = sq.seq0, hi = sq.seq1;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.cu_q[mid] <= tok) lo = mid;
                else hi = mid;
            }
            ctx = min(sq.key1, max(a.context_lens[lo], 0));
        }
        lim_ctx[b] = ctx;
        lim_new[b] = !live ? INT32_MAX : a.block_causal ? min(sq.n_new, (t / a.dbs + 1) * a.dbs) : sq.n_new;
    }
    // Returns whether its rows may see different keys of the tiles [.., u1).
    DFX_D bool start_item(int rows_from, int u1, bool is_group, int pass) {
        lane_off = kvh * static_cast<uint64_t>(a.c_sh) + lane % kChunks * 16;
        table = a.block_tables + sq.table * a.bt_stride;
        const bool uneven = uneven_group(is_group);
        w.reset();
        start_rows(0, rows_from, uneven);
        if constexpr (NB > 1) start_rows(1, rows_from, uneven);
        key_end = is_group && pass >= 0 ? pass : sq.key1;
        new_end = !is_group && pass >= 0 ? pass : sq.n_new;
        return uneven || (a.block_causal && sq.n_new > a.dbs && u1 > sq.ctx_tiles);
    }
    // Hidden keys that are not finite.  A hidden key's weight is 0, but 0 times an infinity or NaN is NaN: in an item whose rows do not
    // all see the same keys (a group with contexts that end inside the prefix, blocks that do not see the later ones) it would spoil rows
    // for which it does not exist.  Nothing in the loops looks for that; where a finished sum of such a row is NaN the item is run again for
    // each number of keys that its rows see, `pass`, with zeros for the others and for the rows that see just these.
    // Returns the next pass, -1: none (the same for all waves).
    DFX_D bool spoilt(bool is_group) const {
        bool nan = false;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) nan |= w.o[d][0][i] != w.o[d][0][i];
        return nan && hides(is_group);
    }
    DFX_D bool hides(bool is_group) const { return is_group ? lim_ctx[0] < sq.key1 : lim_new[0] < sq.n_new; }
    DFX_D bool written(bool is_group, int pass) const { return pass < 0 || (is_group ? lim_ctx[0] : lim_new[0]) == pass; }
    DFX_D int another_pass(bool is_group, int pass, bool any_spoilt) {
        if (pass < 0 && !__syncthreads_or(any_spoilt)) return -1;
        const int limit = is_group ? lim_ctx[0] : lim_new[0];
        int* least = reinterpret_cast<int*>(ml);
        lds_barrier();
        if (tid == 0) *least = INT32_MAX;
        lds_barrier();
        if (hides(is_group) && limit > pass) atomicMin(least, limit);
        lds_barrier();
        const int next = uniform(*least);
        lds_barrier();
        return next == INT32_MAX ? -1 : next;
    }
    DFX_D bool uneven_group(bool is_group) {
        if (!is_group) return false;
        bool any = false;
        for (int s = sq.seq0 + tid; s < sq.seq1; s += kWgThreads) any |= a.context_lens[s] < sq.key1;
        return __syncthreads_or(any);
    }

    DFX_D float* acc_slot(int64_t slot) const { return reinterpret_cast<float*>(a.workspace + a.slot_off + slot * kAccBytes); }
    DFX_D float* ml_slot(int64_t slot) const { return reinterpret_cast<float*>(a.workspace + a.ml_off) + slot * 64; }
    DFX_D bool has_slot(int64_t slot) const { return slot < a.first_slot[WIDE] + a.n_slots[WIDE]; }

    // d block `d` of the row block from row rows_from on: a piece to its slot, or the finished rows to the output.
    DFX_D void put(f32x16 o, int d, float inv, int rows_from, int64_t slot, bool direct, bool mine) {
        const int row = rows_from + w.col;
        if (row >= sq.rows || !mine) return;
        if (direct) {
            const int t = row / a.group_heads, g = row - t * a.group_heads;
            uint16_t* dst = a.out + (sq.tok0 + static_cast<int64_t>(t)) * a.o_st + (static_cast<int64_t>(kvh) * a.group_heads + g) * a.o_sh;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                u32x2 r;
                r.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{o[4 * x] * inv, o[4 * x + 1] * inv}, bf16x2));
                r.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{o[4 * x + 2] * inv, o[4 * x + 3] * inv}, bf16x2));
                *reinterpret_cast<u32x2*>(dst + d * 32 + x * 8 + w.half * 4) = r;
            }
        } else {
            f32x4* p = reinterpret_cast<f32x4*>(acc_slot(slot));
#pragma unroll
            for (int x = 0; x < 4; ++x) p[(d * 4 + x) * 64 + lane] = f32x4{o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]};
        }
    }

    // ---- wide ----------------------------------------------------------------------------------
    // Context tiles, in two half steps each: (1) the weights of tile u from its scores, and beside them the scores of tile u + 1;
    // (2) the outputs of tile u, and the wave's share of K of u + 3 and V of u + 2 from registers to LDS and of the tiles behind
    // them from memory to registers.  The first is bound by the exponentials, the second by the matrix pipeline and by moving data:
    // waves 4 to 7, which share their SIMDs with waves 0 to 3, run half a step behind, so that each SIMD has one wave in either.  (In step,
    // the first half took 2100 cycles of a tile's 5100 and the wait at the barrier 1100.)
    // What a half step reads was written two barriers before, and what it overwrites was read two barriers before, by the waves of
    // either half: three buffers of K (scores of u + 1, u + 2, the one being written) and three of V.
    // No branch on the tile's kind in the loop and every wait for a step's loads before the next are issued: where a wait can be reached
    // with other loads in flight, the compiler waits for all of them.
    DFX_D int wide(int u0, int u1, bool is_group, int64_t slot, bool direct, int pass) {
        const int rows_from = row_tile * kWideRows + wave * 32;
        const bool mixed = start_item(rows_from, u1, is_group, pass);
        const bool busy = rows_from < sq.rows;
        const int r0 = wave * ROWS;
        const int c1 = min(u1, sq.ctx_tiles);
        if (u0 < c1) {
            Stage sk, sv;
            f32x16 s[2][NB];
            float top[NB];
            Place at3;                                // of tile u + 3
            Key key4;                                 // keys of tile u + 4
            uint64_t valid0, valid1, valid2, valid3;  // keys with a cache row of tiles u, u + 1, ...
            uint8_t *ka = lds, *kb = lds + kMat, *kc = lds + 2 * kMat;                  // K of u + 3 (and u), u + 1, u + 2
            uint8_t *va = lds + 3 * kMat, *vb = lds + 4 * kMat, *vc = lds + 5 * kMat;  // V of u, u + 1, u + 2
            {
                const Key key0 = look_up(u0), key1 = look_up(u0 + 1), key2 = look_up(u0 + 2), key3 = look_up(u0 + 3);
                key4 = look_up(u0 + 4);
                const Place at0 = place_of(row_of(key0, valid0), r0), at1 = place_of(row_of(key1, valid1), r0);
                const Place at2 = place_of(row_of(key2, valid2), r0);
                at3 = place_of(row_of(key3, valid3), r0);
                Stage k1, k2, v1;
                issue(sk, a.k_cache, a.k_scales, at0);
                issue(k1, a.k_cache, a.k_scales, at1);
                issue(sv, a.v_cache, a.v_scales, at0);
                issue(k2, a.k_cache, a.k_scales, at2);
                issue(v1, a.v_cache, a.v_scales, at1);
                commit(sk, ka, r0, valid0);
                commit(k1, kb, r0, valid1);
                commit(sv, va, r0, valid0);
                commit(k2, kc, r0, valid2);
                commit(v1, vb, r0, valid1);
                issue(sv, a.v_cache, a.v_scales, at2);
                issue(sk, a.k_cache, a.k_scales, at3);
            }
            lds_barrier();
            if (busy) {
                w.scores(address(ka), s);
                mask_context(s, u0, valid0);
                top[0] = W::half_max(w.top_of(s, 0)) * a.c;
            }
            lds_barrier();
            const bool behind = wave >= kWgWaves / 2;
            if (behind) lds_barrier();
            for (int u = u0; u + 1 < c1; ++u) {
                bf16x8 p[NB][2][2];
                f32x16 next[2][NB];
                const Key key5 = look_up(u + 5);
                if (busy) {
                    w.raise(0, top[0]);
                    w.weights_and_scores(s, a.c, p, address(kb), next);
                    mask_context(next, u + 1, valid1);
                }
                lds_barrier();
                if (busy) {
                    w.accumulate_and_top(address(va), p, next, top);
                    top[0] = W::half_max(top[0]) * a.c;
                    s[0][0] = next[0][0];
                    s[1][0] = next[1][0];
                }
                uint64_t valid4;
                const Place at4 = place_of(row_of(key4, valid4), r0);
                commit(sv, vc, r0, valid2);  // (of tiles u + 2 and u + 3; behind the last, zeros that nobody reads)
                commit(sk, ka, r0, valid3);
                issue(sv, a.v_cache, a.v_scales, at3);
                at3 = at4;
                issue(sk, a.k_cache, a.k_scales, at3);
                valid1 = valid2;
                valid2 = valid3;
                valid3 = valid4;
                key4 = key5;
                uint8_t* const k_old = ka;
                uint8_t* const v_old = va;
                ka = kb, kb = kc, kc = k_old;
                va = vb, vb = vc, vc = v_old;
                lds_barrier();
            }
            if (busy) {
                bf16x8 p[NB][2][2];
                w.raise(0, top[0]);
                w.weights(s, a.c, p);
                w.accumulate(address(va), p);
            }
            if (!behind) lds_barrier();
        }
        for (int u = max(u0, sq.ctx_tiles); u < u1; ++u) {
            const int t = u - sq.ctx_tiles;
            lds_barrier();
            fresh_rows(a.k_new, a.kn_st, a.kn_sh, t, lds, r0);
            fresh_rows(a.v_new, a.vn_st, a.vn_sh, t, lds + kMat, r0);
            lds_barrier();
            if (busy) whole_tile(lds, lds + kMat, [&](auto& s) { mask_fresh(s, t); });
        }
        lds_barrier();  // (the next item's tiles)
        if (busy && (direct || has_slot(slot + wave))) {
            const float l = W::half_sum(w.l[0]);
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
            for (int d = 0; d < NDB; ++d) put(w.o[d][0], d, inv, rows_from, slot + wave, direct, written(is_group, pass));
            if (!direct && written(is_group, pass)) ml_slot(slot + wave)[lane] = w.half ? l : w.m[0];
        }
        return mixed ? another_pass(is_group, pass, spoilt(is_group)) : -1;
    }

    // ---- narrow --------------------------------------------------------------------------------
    DFX_D int narrow(int u0, int u1, bool is_group, int64_t slot, bool direct, int pass) {
        uint8_t* kt = lds + wave * 2 * kMat;
        uint8_t* vt = kt + kMat;
        // wave = head of the group * side + place among the head's waves
        const int side_shift = 2 - a.heads_shift, side = 1 << side_shift;
        const int my_head = wave >> side_shift;
        kvh = (kvh << a.heads_shift) + my_head;
        slot += my_head;
        const bool mixed = start_item(row_tile * kNarrowRows, u1, is_group, pass);
        int u = u0 + (wave & (side - 1));
        const int c1 = min(u1, sq.ctx_tiles);
        if (u < c1) {
            Stage sk[kDepth], sv[kDepth];
            uint64_t valid[kDepth];
            // A table entry is looked up kDepth tiles before its rows' loads are issued, so that it is in front of the loads that a tile's
            // commit waits for: loads return in order, and a wait for a younger entry would drain the tiles in flight (as reloads of spilled
            // registers do: see kDepth).
            Key keys[kDepth];
#pragma unroll
            for (int i = 0; i < kDepth; ++i) keys[i] = look_up(u + i * side);
#pragma unroll
            for (int i = 0; i < kDepth; ++i) {
                const Place at = place_of(row_of(keys[i], valid[i]), 0);
                keys[i] = look_up(u + (kDepth + i) * side);
                issue(sk[i], a.k_cache, a.k_scales, at);
                issue(sv[i], a.v_cache, a.v_scales, at);
            }
            auto step = [&](Stage& k, Stage& v, uint64_t& v_of, Key& key) {
                commit(k, kt, 0, v_of);
                commit(v, vt, 0, v_of);
                const uint64_t here = v_of;
                const Place at = place_of(row_of(key, v_of), 0);
                key = look_up(u + 2 * kDepth * side);
                issue(k, a.k_cache, a.k_scales, at);
                issue(v, a.v_cache, a.v_scales, at);
                asm volatile("" ::: "memory");  // (the tile is the wave's own: LDS keeps the wave's order)
                whole_tile(kt, vt, [&](auto& s) { mask_context(s, u, here); });
                asm volatile("" ::: "memory");
                u += side;
                return u < c1;
            };
            for (;;) {  // (written out: a loop over the stages that is left in the middle is not unrolled)
                if (!step(sk[0], sv[0], valid[0], keys[0])) break;
                if constexpr (kDepth > 1)
                    if (!step(sk[1], sv[1], valid[1], keys[1])) break;
                if constexpr (kDepth > 2)
                    if (!step(sk[2], sv[2], valid[2], keys[2])) break;
                static_assert(kDepth <= 3, "one step per stage");
            }
        }
        for (; u < u1; u += side) {
            const int t = u - sq.ctx_tiles;
            fresh_rows(a.k_new, a.kn_st, a.kn_sh, t, kt, 0);
            fresh_rows(a.v_new, a.vn_st, a.vn_sh, t, vt, 0);
            asm volatile("" ::: "memory");
            whole_tile(kt, vt, [&](auto& s) { mask_fresh(s, t); });
            asm volatile("" ::: "memory");
        }
        const float l = W::half_sum(w.l[0]);
        if (side == 1) {
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            if (direct || has_slot(slot)) {
#pragma unroll
                for (int d = 0; d < NDB; ++d) put(w.o[d][0], d, inv, row_tile * kNarrowRows, slot, direct, written(is_group, pass));
                if (!direct && written(is_group, pass)) ml_slot(slot)[lane] = w.half ? l : w.m[0];
            }
            return mixed ? another_pass(is_group, pass, spoilt(is_group)) : -1;
        }
        // merge the states of a head's waves: each leaves its accumulators in its own LDS, and takes every side-th d block
        ml[wave * 64 + lane] = w.half ? l : w.m[0];
        f32x4* mine = reinterpret_cast<f32x4*>(lds + wave * kAccBytes);
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                mine[(d * 4 + x) * 64 + lane] = f32x4{w.o[d][0][4 * x], w.o[d][0][4 * x + 1], w.o[d][0][4 * x + 2], w.o[d][0][4 * x + 3]};
        lds_barrier();
        const int from = my_head << side_shift;
        float top = -INFINITY, sum = 0.0f;
        for (int i = from; i < from + side; ++i) top = fmaxf(top, ml[i * 64 + w.col]);
        const float base = top == -INFINITY ? 0.0f : top;
        for (int i = from; i < from + side; ++i) sum += __builtin_amdgcn_exp2f(ml[i * 64 + w.col] - base) * ml[i * 64 + 32 + w.col];
        const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
        for (int d = wave & (side - 1); d < NDB; d += side) {
            f32x16 o;
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0.0f;
            for (int i = from; i < from + side; ++i) {
                const float f = __builtin_amdgcn_exp2f(ml[i * 64 + w.col] - base);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const f32x4 p = reinterpret_cast<const f32x4*>(lds + i * kAccBytes)[(d * 4 + x) * 64 + lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[4 * x + j] += f * p[j];
                }
            }
            if (direct || has_slot(slot)) put(o, d, inv, row_tile * kNarrowRows, slot, direct, written(is_group, pass));
        }
        if (!direct && (wave & (side - 1)) == 0 && has_slot(slot) && written(is_group, pass)) ml_slot(slot)[lane] = w.half ? sum : top;
        lds_barrier();
        return mixed ? another_pass(is_group, pass, spoilt(is_group)) : -1;
    }
};

struct Sums {
    int64_t cost;      // of the launch's kind
    int blocks, comb;  // piece slots of its items; row blocks of the merge
    DFX_D void operator+=(const Sums& o) {
        cost += o.cost;
        blocks += o.blocks;
        comb += o.comb;
    }
};
template <bool WIDE>
DFX_D Sums sums_of(const SplitArgs& a, const Seq& s, int v) {
    const Costs k(a, !WIDE);
    const int items = s.narrow != WIDE ? a.h_kv / k.heads * s.row_tiles : 0;
    return Sums{static_cast<int64_t>(items) * item_cost(k, s.tiles), items * k.blocks, v >= a.n_groups ? a.h_kv * ((s.rows + 31) / 32) : 0};
}
DFX_D Sums lane_below(Sums v, int by) {
    const int from = static_cast<int>(threadIdx.x & 63) - by;
    const int at = (from < 0 ? 0 : from) * 4;
    const int lo = __builtin_amdgcn_ds_bpermute(at, static_cast<int>(v.cost)), hi = __builtin_amdgcn_ds_bpermute(at, static_cast<int>(v.cost >> 32));
    Sums r;
    r.cost = static_cast<int64_t>(static_cast<uint32_t>(lo)) | (static_cast<int64_t>(hi) << 32);
    r.blocks = __builtin_amdgcn_ds_bpermute(at, v.blocks);
    r.comb = __builtin_amdgcn_ds_bpermute(at, v.comb);
    return from < 0 ? Sums{0, 0, 0} : r;
}

DFX_D Seq uniform_seq(const Seq& s) {  // (what LDS returns is a vector register to the compiler)
    return Seq{uniform(s.tok0), uniform(s.rows), uniform(s.key0), uniform(s.key1), uniform(s.new0), uniform(s.n_new), uniform(s.table),
               uniform(s.prefix), uniform(s.seq0), uniform(s.seq1), uniform(s.tiles), uniform(s.ctx_tiles), uniform(s.row_tiles),
               uniform(s.narrow) != 0, uniform(s.group)};
}

// Number of the i-th of `launched` workgroups among the `n_wg` that work (n_wg or more: none).  Workgroups go to the eight XCDs in turn: neighbouring
// ranges (the row tiles that read the same keys) are to be on one of them.
DFX_D int numbered(int i, int launched, int n_wg) {
    const int xcd = i % 8, slot = i / 8, each = launched / 8;
    if (n_wg > each * 8) return xcd * each + min(xcd, launched % 8) + slot;  // (all of them, the last round of the XCDs is not full)
    const int used = (n_wg + 7) / 8;
    return slot < used ? xcd * used + slot : n_wg;
}

template <int HD, int KV, bool WIDE>
__global__ void __launch_bounds__(Kind<WIDE>::kThreads, 2) split_attn_kernel(const SplitArgs a) {
    using T = Split<HD, KV, WIDE>;
    constexpr int kWgWaves = Kind<WIDE>::kWaves, kWgThreads = Kind<WIDE>::kThreads;
    __shared__ __attribute__((aligned(256))) uint8_t lds[T::kLds];
    __shared__ float ml[kWgWaves * 64];
    __shared__ Sums wave_sum[kWgWaves];
    __shared__ int first_v, first_blocks;
    __shared__ int64_t first_cost;
    __shared__ Seq first_seq;
    const int tid = threadIdx.x;

    // the work list: each thread a run of virtual sequences, then a scan
    const int n = a.n_groups + a.n_seqs;
    const int per = (n + kWgThreads - 1) / kWgThreads;
    const Costs kinds(a, !WIDE);
    const Seq my_first = seq_of(a, min(tid * per, n - 1));  // (with up to a virtual sequence per thread, read once)
    auto seq_at = [&](int i) { return i == 0 ? my_first : seq_of(a, tid * per + i); };
    Sums mine = {0, 0, 0};
    for (int i = 0; i < per; ++i) {
        const int v = tid * per + i;
        if (v >= n) break;
        mine += sums_of<WIDE>(a, seq_at(i), v);
    }
    Sums upto = mine;
#pragma unroll
    for (int by = 1; by < 64; by *= 2) upto += lane_below(upto, by);
    if ((tid & 63) == 63) wave_sum[tid >> 6] = upto;
    __syncthreads();
    Sums total = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < kWgWaves; ++i) {
        if (i < (tid >> 6)) upto += wave_sum[i];
        total += wave_sum[i];
    }
    int n_wg = a.n_wg[WIDE];
    if (total.cost / kinds.least < n_wg) n_wg = static_cast<int>(max(total.cost / kinds.least, static_cast<int64_t>(1)));
    if (blockIdx.x == 0) {  // the list, for the merge; the others work
        if (tid == 0) reinterpret_cast<Header*>(a.workspace)[WIDE] = Header{total.cost, n_wg, total.comb};
        Sums at = {upto.cost - mine.cost, upto.blocks - mine.blocks, upto.comb - mine.comb};
        int* comb = reinterpret_cast<int*>(a.workspace + a.comb_off);
        for (int i = 0; i < per; ++i) {
            const int v = tid * per + i;
            if (v >= n) break;
            const Seq s = seq_at(i);
            if (s.narrow != WIDE)
                reinterpret_cast<Rec*>(a.workspace + a.rec_off)[v] =
                    Rec{at.cost, at.blocks, s.tok0, s.rows, s.tiles, s.row_tiles, s.prefix > 0 ? s.group : -1, s.narrow, s.key1 > 0 || s.n_new > 0};
            if (!WIDE && v >= a.n_groups) comb[v - a.n_groups] = at.comb;
            at += sums_of<WIDE>(a, s, v);
        }
        if (!WIDE && tid == 0) comb[a.n_seqs] = total.comb;
        return;
    }
    const int wg = numbered(static_cast<int>(blockIdx.x - 1), a.n_wg[WIDE], n_wg);
    if (wg >= n_wg || total.cost == 0) return;
    const int64_t c0 = range_start(wg, total.cost, n_wg), c1 = range_start(wg + 1, total.cost, n_wg);
    if (c0 >= c1) return;
    if (upto.cost > c0 && upto.cost - mine.cost <= c0) {  // this thread's run holds the first unit
        Sums at = {upto.cost - mine.cost, upto.blocks - mine.blocks, 0};
        for (int i = 0; i < per; ++i) {
            const int v = tid * per + i;
            const Seq s = seq_at(i);
            const Sums here = sums_of<WIDE>(a, s, v);
            if (at.cost + here.cost > c0) {
                first_v = v;
                first_cost = at.cost;
                first_blocks = at.blocks;
                first_seq = s;
                break;
            }
            at += here;
        }
    }
    __syncthreads();
    int64_t cost = first_cost;
    cost = static_cast<int64_t>(static_cast<uint32_t>(uniform(static_cast<int>(cost)))) | (static_cast<int64_t>(uniform(static_cast<int>(cost >> 32))) << 32);
    int blocks = uniform(first_blocks);
    T t(a, lds, ml, tid);
    t.sq = uniform_seq(first_seq);
    for (int v = uniform(first_v);;) {
        const Seq& s = t.sq;
        if (s.narrow != WIDE) {
            const int items = a.h_kv / kinds.heads * s.row_tiles, each = item_cost(kinds, s.tiles);
            if (each > 0) {
                int j = cost < c0 ? static_cast<int>((c0 - cost) / each) : 0;
                int pass = -1;
                for (; j < items; j += pass < 0) {
                    const int64_t from = cost + static_cast<int64_t>(j) * each;
                    if (from >= c1) break;
                    const int u0 = from >= c0 ? 0 : static_cast<int>(c0 - from);
                    const int u1 = static_cast<int>(min(static_cast<int64_t>(s.tiles), c1 - from));
                    if (u0 >= u1) continue;
                    const int head = j / s.row_tiles;  // or group of heads
                    t.kvh = head;
                    t.row_tile = j - head * s.row_tiles;
                    const bool is_group = v < a.n_groups;
                    const bool direct = !is_group && s.prefix == 0 && u0 == 0 && u1 == s.tiles;
                    const int64_t slot = a.first_slot[WIDE] + (static_cast<int64_t>(wg) + j) * kinds.blocks + blocks;
                    if constexpr (WIDE) pass = t.wide(u0, u1, is_group, slot, direct, pass);
                    else pass = t.narrow(u0, u1, is_group, slot, direct, pass);
                }
            }
            cost += static_cast<int64_t>(items) * each;
            blocks += items * kinds.blocks;
        }
        if (++v >= n || cost >= c1) break;
        t.sq = seq_of(a, v);
    }
}

// ---- merge -------------------------------------------------------------------------------------
// One workgroup per (sequence, KV head, 32 rows): NDB waves for the d blocks, times kShare that take every kShare-th piece of the row,
// kAtOnce of them together.  Bound by latency: the list and the pieces lie in memory that another XCD wrote, so everything that may be
// needed of the list is asked for at once.  (The order of the sums is the pieces', whoever finished first.)
constexpr int kAtOnce = 4;
// Few row blocks have many pieces each (the work is spread over all workgroups), many have few.  (Whole calls with 4 and with 16 waves, us: 256 blocks 43,
// 34; 800 blocks 56, 61; 2048 blocks 80, 102.)
constexpr int kMergeWavesFew = 16, kMergeWavesMany = 4, kFewBlocks = 512;

template <int HD, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) split_merge_kernel(const SplitArgs a) {
    constexpr int NDB = HD / 32, kShare = WAVES / NDB;
    constexpr int kAccBytes = 32 * HD * 4;
    __shared__ int found_at;
    __shared__ Rec found_rec, group_rec;
    __shared__ float part[kShare > 1 ? WAVES : 1][18][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, half = lane >> 5;
    const Header* heads = reinterpret_cast<const Header*>(a.workspace);
    const int x = blockIdx.x;
    const int* comb = reinterpret_cast<const int*>(a.workspace + a.comb_off);
    const Rec* recs = reinterpret_cast<const Rec*>(a.workspace + a.rec_off);
    const Header head_of[2] = {heads[0], heads[1]};
    const Rec my_group = recs[min(tid, a.n_groups)];
    for (int s = tid; s < a.n_seqs; s += WAVES * 64) {
        const int from = comb[s], to = comb[s + 1];
        const Rec r = recs[a.n_groups + s];
        if (from <= x && x < to) {
            found_at = from;
            found_rec = r;
        }
    }
    if (x >= head_of[0].n_comb) return;
    __syncthreads();
    const Rec q = found_rec;
    if (!q.has_keys) return;  // no key at all: the rows stay as they are
    const int rbs = (q.rows + 31) / 32;
    const int local = x - found_at, kvh = local / rbs, rb = local - kvh * rbs;
    const int row = rb * 32 + col;
    const bool live = row < q.rows;

    // the pieces of this lane's row: its own item's, then its group's.  slot of piece i: first + i * step
    int64_t first[2] = {0, 0};
    int n[2] = {0, 0}, at_col[2] = {col, 0}, step[2] = {1, 1};
    auto pieces = [&](const Rec& r, int k, int at_row) {
        const Header h = r.narrow ? head_of[0] : head_of[1];
        const Costs c(a, r.narrow);
        const int most = r.narrow ? kNarrowRows : kWideRows, t = at_row / most;
        const int64_t j = static_cast<int64_t>(kvh / c.heads) * r.row_tiles + t, from = r.cost + j * item_cost(c, r.tiles);
        const int w0 = owner_of(from, h.total, h.n_wg);
        n[k] = owner_of(from + r.tiles - 1, h.total, h.n_wg) - w0 + 1;
        first[k] = a.first_slot[r.narrow ? 0 : 1] + (w0 + j) * c.blocks + r.blocks + (r.narrow ? kvh % c.heads : (at_row - t * most) / 32);
        step[k] = c.blocks;
        at_col[k] = at_row & 31;
    };
    if (q.tiles > 0) {
        pieces(q, 0, rb * 32);
        at_col[0] = col;
        if (q.group < 0 && n[0] == 1) return;  // written by its only workgroup
    }
    if (q.group >= 0) {
        if (a.n_groups < WAVES * 64) {
            if (tid == q.group) group_rec = my_group;
        } else if (tid == 0) {
            group_rec = recs[q.group];
        }
        __syncthreads();
        const Rec g = group_rec;
        if (g.tiles > 0) pieces(g, 1, max(0, (q.tok0 - g.tok0) * a.group_heads + (live ? row : 0)));
    }
    const int d = wave % NDB, share = wave / NDB;
    float m = -INFINITY, l = 0.0f;
    f32x4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = f32x4{0, 0, 0, 0};
    const int all = live ? n[0] + n[1] : 0;
    const int64_t slots = a.first_slot[1] + a.n_slots[1];
    for (int i0 = share; __builtin_amdgcn_ballot_w64(i0 < all) != 0; i0 += kShare * kAtOnce) {
        float pm[kAtOnce], pl[kAtOnce];
        f32x4 po[kAtOnce][4];
#pragma unroll
        for (int y = 0; y < kAtOnce; ++y) {
            const int i = i0 + y * kShare;
            const bool mine = i < n[0];
            const int64_t slot = mine ? first[0] + static_cast<int64_t>(i) * step[0] : first[1] + static_cast<int64_t>(i - n[0]) * step[1];
            const int c = mine ? at_col[0] : at_col[1];
            const bool is = i < all && slot >= 0 && slot < slots;
            const float* ml = reinterpret_cast<const float*>(a.workspace + a.ml_off) + (is ? slot : 0) * 64;
            const f32x4* acc = reinterpret_cast<const f32x4*>(a.workspace + a.slot_off + (is ? slot : 0) * kAccBytes);
            pm[y] = -INFINITY;
            pl[y] = 0.0f;
#pragma unroll
            for (int z = 0; z < 4; ++z) po[y][z] = f32x4{0, 0, 0, 0};
            if (is) {
                pm[y] = ml[c];
                pl[y] = ml[32 + c];
#pragma unroll
                for (int z = 0; z < 4; ++z) po[y][z] = acc[(d * 4 + z) * 64 + half * 32 + c];
            }
        }
        float top = m;
#pragma unroll
        for (int y = 0; y < kAtOnce; ++y) top = fmaxf(top, pm[y]);
        const float base = top == -INFINITY ? 0.0f : top;  // (pieces without a visible key: weight 2^-inf = 0 of zeros)
        const float keep = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l *= keep;
#pragma unroll
        for (int z = 0; z < 4; ++z) o[z] *= keep;
#pragma unroll
        for (int y = 0; y < kAtOnce; ++y) {
            const float f = __builtin_amdgcn_exp2f(pm[y] - base);
            l += pl[y] * f;
#pragma unroll
            for (int z = 0; z < 4; ++z) o[z] += po[y][z] * f;
        }
    }
    if constexpr (kShare > 1) {
        if (share > 0) {
            part[wave][0][lane] = m;
            part[wave][1][lane] = l;
#pragma unroll
            for (int y = 0; y < 16; ++y) part[wave][2 + y][lane] = o[y >> 2][y & 3];
        }
        __syncthreads();
        if (share > 0) return;
#pragma unroll
        for (int i = 1; i < kShare; ++i) {
            const int other = wave + i * NDB;
            const float pm = part[other][0][lane], pl = part[other][1][lane];
            const float top = fmaxf(m, pm), base = top == -INFINITY ? 0.0f : top;
            const float keep = __builtin_amdgcn_exp2f(m - base), add = __builtin_amdgcn_exp2f(pm - base);
            m = top;
            l = l * keep + pl * add;
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y >> 2][y & 3] = o[y >> 2][y & 3] * keep + part[other][2 + y][lane] * add;
        }
    }
    if (!live) return;
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const int t = row / a.group_heads, g = row - t * a.group_heads;
    uint16_t* dst = a.out + (q.tok0 + static_cast<int64_t>(t)) * a.o_st + (static_cast<int64_t>(kvh) * a.group_heads + g) * a.o_sh;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
        u32x2 r;
        r.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{o[y][0] * inv, o[y][1] * inv}, bf16x2));
        r.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{o[y][2] * inv, o[y][3] * inv}, bf16x2));
        *reinterpret_cast<u32x2*>(dst + d * 32 + y * 8 + half * 4) = r;
    }
}

int compute_units() {
    static int cached[64] = {0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -1;
    if (cached[dev] == 0) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return -1;
        cached[dev] = n;
    }
    return cached[dev];
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Sizes of the launches and of their workspace; a status.
int lay_out(const dfx_split_attn_params* p, SplitArgs& a, int64_t& comb_blocks, int64_t& bytes) {
    if (!p || p->num_seqs < 0 || p->num_groups < 0 || p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->num_q_tokens < 0 ||
        p->num_new_tokens < 0 || p->max_workgroups < 0 || p->max_seqlen_q < 0)
        return DFX_ERR_INVALID_ARG;
    if (p->num_q_heads % p->num_kv_heads != 0) return DFX_ERR_INVALID_ARG;
    if (p->head_dim != 64 && p->head_dim != 128) return DFX_ERR_UNSUPPORTED;
    if (p->num_seqs > 65535 || p->num_groups > p->num_seqs + 1 || p->num_q_tokens > INT32_MAX / p->num_q_heads ||
        p->num_new_tokens > INT32_MAX || p->max_workgroups > 65535)
        return DFX_ERR_UNSUPPORTED;
    a.n_wg[0] = a.n_wg[1] = p->max_workgroups;
    if (p->max_workgroups == 0) {  // what the device holds at once, the list's workgroup included
        const int cus = compute_units();
        if (cus < 0) return DFX_ERR_LAUNCH;
        a.n_wg[0] = 2 * cus - 1;
        a.n_wg[1] = cus - 1 > 0 ? cus - 1 : 1;
    }
    a.n_seqs = p->num_seqs;
    a.n_groups = p->num_groups;
    a.h_kv = p->num_kv_heads;
    a.group_heads = p->num_q_heads / p->num_kv_heads;
    // rows of the largest virtual sequence, as far as the host knows: without wide items there is no wide launch
    const int64_t rows = p->num_q_tokens * a.group_heads;
    int64_t most = p->max_seqlen_q > 0 ? static_cast<int64_t>(p->max_seqlen_q) * a.group_heads : rows;
    if (most > rows || p->num_groups > 0) most = rows;
    a.use_wide = most > kNarrowMost;
    const int64_t rows32 = (rows + 31) / 32, vs = static_cast<int64_t>(p->num_seqs) + p->num_groups;
    comb_blocks = a.h_kv * (rows32 + p->num_seqs);
    // (an item of R rows takes at most R / 32 + 1 slots if it is narrow, R / 32 + 8 if it is wide, which needs more than kNarrowMost rows)
    const int64_t copies = (p->num_groups > 0 ? 2 : 1) * rows32;
    const int64_t wide_vs = vs < copies * 32 / kNarrowMost ? vs : copies * 32 / kNarrowMost;
    a.heads_shift = a.h_kv % 4 == 0 ? 2 : a.h_kv % 2 == 0 ? 1 : 0;
    // (a piece's slot is the sum of its workgroup's and its item's index)
    a.n_slots[0] = (static_cast<int64_t>(a.n_wg[0]) << a.heads_shift) + a.h_kv * (copies + vs);
    a.n_slots[1] = a.use_wide ? (a.n_wg[1] + a.h_kv * wide_vs) * (kWideRows / 32) + a.h_kv * copies : 0;
    a.first_slot[0] = 0;
    a.first_slot[1] = a.n_slots[0];
    const int64_t slots = a.n_slots[0] + a.n_slots[1];
    if (comb_blocks > UINT32_MAX / (kMergeWavesFew * 64) || slots > INT32_MAX) return DFX_ERR_UNSUPPORTED;
    a.rec_off = 256;
    a.comb_off = a.rec_off + round_up(vs * static_cast<int64_t>(sizeof(Rec)), 256);
    a.ml_off = a.comb_off + round_up((static_cast<int64_t>(p->num_seqs) + 1) * 4, 256);
    a.slot_off = a.ml_off + slots * 256;
    bytes = a.slot_off + slots * 32 * p->head_dim * 4;
    return DFX_OK;
}

}  // namespace
}  // namespace dfx

using namespace dfx;

extern "C" int64_t dfx_split_attn_workspace_bytes(const dfx_split_attn_params* p) {
    SplitArgs a{};
    int64_t comb = 0, bytes = 0;
    const int rc = lay_out(p, a, comb, bytes);
    return rc == DFX_OK ? bytes : rc;
}

extern "C" int dfx_split_attn(const dfx_split_attn_params* p, dfx_stream_t stream) {
    SplitArgs a{};
    int64_t comb = 0, bytes = 0;
    const int rc = lay_out(p, a, comb, bytes);
    if (rc != DFX_OK) return rc;
    if (p->num_seqs == 0 || p->num_q_tokens == 0) return DFX_OK;
    const bool mx = p->kv_dtype == DFX_KV_MX_E4M3 || p->kv_dtype == DFX_KV_MX_E2M1;
    if (!mx && p->kv_dtype != DFX_KV_BF16) return DFX_ERR_INVALID_ARG;
    if (p->mask_mode != DFX_MASK_FULL && p->mask_mode != DFX_MASK_BLOCK_CAUSAL) return DFX_ERR_INVALID_ARG;
    if (p->mask_mode == DFX_MASK_BLOCK_CAUSAL && p->diffusion_block_size <= 0) return DFX_ERR_INVALID_ARG;
    if (!(p->scale > 0.0f) || !(p->scale < INFINITY)) return DFX_ERR_INVALID_ARG;
    if (!p->q || !p->out || !p->cu_seqlens_q || !p->cu_seqlens_new) return DFX_ERR_INVALID_ARG;
    if (p->num_new_tokens > 0 && (!p->k_new || !p->v_new)) return DFX_ERR_INVALID_ARG;
    if (p->num_groups > 0 && (!p->prefix_cu_seqs || !p->prefix_lens || !p->k_cache)) return DFX_ERR_INVALID_ARG;
    const void* aligned[] = {p->q, p->out, p->k_new, p->v_new, p->k_cache, p->v_cache};
    for (const void* x : aligned)
        if (!aligned16(x)) return DFX_ERR_INVALID_ARG;
    const int64_t strides[] = {p->q_stride_token, p->q_stride_head, p->kn_stride_token, p->kn_stride_head, p->vn_stride_token, p->vn_stride_head,
                               p->o_stride_token, p->o_stride_head};
    for (int64_t s : strides)
        if (s % 8 || s < 0) return DFX_ERR_INVALID_ARG;
    const bool cached = p->k_cache && p->n_pages != 0 && p->max_pages_per_seq != 0;
    if (cached) {
        if (!p->v_cache || !p->block_tables || !p->context_lens || p->page_size <= 0 || p->n_pages < 0 || p->max_pages_per_seq < 0 ||
            p->block_table_stride < 0)
            return DFX_ERR_INVALID_ARG;
        if (mx != (p->k_scales != nullptr) || mx != (p->v_scales != nullptr)) return DFX_ERR_INVALID_ARG;
        if (p->n_pages > INT32_MAX) return DFX_ERR_UNSUPPORTED;
        int64_t page_bytes, token_bytes, head_bytes;
        if (mx) {
            head_bytes = mx_row_bytes(p->kv_dtype == DFX_KV_MX_E2M1, p->head_dim);
            token_bytes = head_bytes * p->num_kv_heads;
            page_bytes = token_bytes * p->page_size;
        } else {
            if (p->cache_stride_page % 8 || p->cache_stride_token % 8 || p->cache_stride_head % 8 || p->cache_stride_page < 0 ||
                p->cache_stride_token < 0 || p->cache_stride_head < 0)
                return DFX_ERR_INVALID_ARG;
            page_bytes = p->cache_stride_page * 2;
            token_bytes = p->cache_stride_token * 2;
            head_bytes = p->cache_stride_head * 2;
        }
        if (page_bytes > UINT32_MAX || token_bytes > UINT32_MAX || head_bytes > UINT32_MAX) return DFX_ERR_UNSUPPORTED;
        a.c_sp = static_cast<uint32_t>(page_bytes);
        a.c_st = static_cast<uint32_t>(token_bytes);
        a.c_sh = static_cast<uint32_t>(head_bytes);
        a.block_tables = p->block_tables;
        a.context_lens = p->context_lens;
        a.bt_stride = p->block_table_stride;
        a.n_pages = static_cast<int>(p->n_pages);
        a.max_pages = p->max_pages_per_seq;
        a.page_size = p->page_size;
        a.page_shift = (p->page_size & (p->page_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(p->page_size)) : -1;
    } else {
        // No cache: no context and no prefix.  The kernel's loads are not conditional -- a key without a cache row loads the first row of
        // the cache and drops it, a tile behind the last its table row's last entry --, they read the workspace here.
        a.page_size = a.max_pages = 1;
        a.block_tables = static_cast<const int32_t*>(p->workspace);
        a.n_groups = 0;
    }
    if (!p->workspace || p->workspace_bytes < bytes) return DFX_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(p->workspace) % 256) return DFX_ERR_INVALID_ARG;
    a.q = static_cast<const uint16_t*>(p->q);
    a.k_new = static_cast<const uint16_t*>(p->k_new);
    a.v_new = static_cast<const uint16_t*>(p->v_new);
    a.out = static_cast<uint16_t*>(p->out);
    a.k_cache = static_cast<const uint8_t*>(cached ? p->k_cache : p->workspace);
    a.v_cache = static_cast<const uint8_t*>(cached ? p->v_cache : p->workspace);
    a.k_scales = static_cast<const uint8_t*>(p->k_scales);
    a.v_scales = static_cast<const uint8_t*>(p->v_scales);
    a.cu_q = p->cu_seqlens_q;
    a.cu_new = p->cu_seqlens_new;
    a.group_cu = p->prefix_cu_seqs;
    a.group_len = p->prefix_lens;
    a.workspace = static_cast<uint8_t*>(p->workspace);
    a.q_st = p->q_stride_token;
    a.q_sh = p->q_stride_head;
    a.kn_st = p->kn_stride_token;
    a.kn_sh = p->kn_stride_head;
    a.vn_st = p->vn_stride_token;
    a.vn_sh = p->vn_stride_head;
    a.o_st = p->o_stride_token;
    a.o_sh = p->o_stride_head;
    a.n_q = static_cast<int>(p->num_q_tokens);
    a.n_new = static_cast<int>(p->num_new_tokens);
    a.dbs = p->diffusion_block_size;
    a.block_causal = p->mask_mode == DFX_MASK_BLOCK_CAUSAL;
    a.c = p->scale * 1.4426950408889634f;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int kv = !cached || !mx ? kBf16 : p->kv_dtype == DFX_KV_MX_E4M3 ? kMx8 : kMx4;
#define DFX_SPLIT_KIND(HD_, WIDE_)                                                                          \
    do {                                                                                                    \
        auto kern = kv == kBf16  ? split_attn_kernel<HD_, kBf16, WIDE_>                                     \
                    : kv == kMx8 ? split_attn_kernel<HD_, kMx8, WIDE_>                                      \
                                 : split_attn_kernel<HD_, kMx4, WIDE_>;                                     \
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(a.n_wg[WIDE_]) + 1), dim3(Kind<WIDE_>::kThreads), 0, st, a);          \
    } while (0)
#define DFX_SPLIT(HD_)                                                                                      \
    do {                                                                                                    \
        if (a.use_wide) DFX_SPLIT_KIND(HD_, true);                                                          \
        DFX_SPLIT_KIND(HD_, false);                                                                         \
        if (comb <= kFewBlocks)                                                                             \
            hipLaunchKernelGGL((split_merge_kernel<HD_, kMergeWavesFew>), dim3(static_cast<unsigned>(comb)), dim3(kMergeWavesFew * 64), 0, st, a); \
        else                                                                                                \
            hipLaunchKernelGGL((split_merge_kernel<HD_, kMergeWavesMany>), dim3(static_cast<unsigned>(comb)), dim3(kMergeWavesMany * 64), 0, st, a); \
    } while (0)
    if (p->head_dim == 128) DFX_SPLIT(128);
    else DFX_SPLIT(64);
#undef DFX_SPLIT
#undef DFX_SPLIT_KIND
    return launch_status();
}
