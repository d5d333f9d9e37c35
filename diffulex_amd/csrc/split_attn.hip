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
// is (virtual sequence, KV head, row tile), a unit one key tile of it; units have a cost and are dealt to the
// workgroups in contiguous ranges of equal cost.  Every workgroup works the list out for itself from the lengths on the device (no
// host read, safe in a captured graph with later lengths); a second launch merges the pieces.
//
// Two item kinds, chosen by the rows:
//   narrow (rows <= 32: single tokens, small blocks): bound by memory.  Each of the four waves takes every fourth
//     32-key tile into LDS of its own (no barrier in the loop, the next tile's loads in flight over the current one's
//     arithmetic) and keeps a softmax state of its own; the four are merged in LDS at the end of the item.
//   wide (more rows): bound by the matrix instructions and their LDS operands.  128 rows, 32 per wave, over 64-key tiles shared
//     by the waves and double buffered.
// Microscaled codes are widened on the way from registers to LDS, once per tile, with their block's scale applied by the same
// instruction: from there on the arithmetic is the bf16 cache's.
#include "attn_tile.h"
#include "mx_format.h"

namespace dfx {
namespace {

constexpr int kWgThreads = 256;
constexpr int kWgWaves = 4;
constexpr int kNarrowRows = 32, kWideRows = 128;
constexpr int kNarrowKeys = 32, kWideKeys = 64;
constexpr int kWideCost = 4;    // cost of a unit: a wide one takes a workgroup about as long as four narrow ones
constexpr int kNarrowCost = 1;
constexpr int kMinCost = 4;     // least cost per workgroup (>= the largest unit's: every range then holds a unit)

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
    int64_t c_sp, c_st, c_sh;  // cache strides in bytes: page, token, head
    int64_t bt_stride;
    int64_t tab_off, comb_off, slot_off, ml_off, n_slots;  // workspace
    int n_pages, n_q, n_new;
    int n_seqs, n_groups, h_kv, group_heads;
    int page_size, page_shift, max_pages, dbs, block_causal, n_wg;
    float c;  // scale * log2(e)
};

struct Header {
    int64_t total;  // cost of all units
    int32_t n_wg;   // workgroups that have work
    int32_t n_comb; // row blocks of the merge
};
struct TabEntry {
    int64_t cost;  // of the units before the virtual sequence
    int32_t blocks;  // row-block slots of the items before it
    int32_t pad;
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
    DFX_D int cost() const { return narrow ? kNarrowCost : kWideCost; }
    DFX_D int row_blocks() const { return narrow ? 1 : kWideRows / 32; }  // slots of an item's piece
};

DFX_D int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Keys of sequence s's context that belong to its group's prefix.
DFX_D int prefix_of(const SplitArgs& a, int s) {
    int lo = 0, hi = a.n_groups;  // the last group that starts at or before s
    if (hi == 0 || s < a.group_cu[0] || s >= a.group_cu[hi]) return 0;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.group_cu[mid] <= s) lo = mid;
        else hi = mid;
    }
    return max(a.group_len[lo], 0);
}

DFX_D Seq seq_of(const SplitArgs& a, int v) {
    Seq q;
    const int64_t capacity = static_cast<int64_t>(a.max_pages) * a.page_size;
    const int cap = static_cast<int>(capacity > INT32_MAX - 64 ? INT32_MAX - 64 : capacity);
    q.new0 = q.n_new = 0;
    if (v < a.n_groups) {
        q.seq0 = clampi(a.group_cu[v], 0, a.n_seqs);
        q.seq1 = clampi(a.group_cu[v + 1], q.seq0, a.n_seqs);
        q.key0 = 0;
        q.key1 = q.prefix = clampi(a.group_len[v], 0, cap);
    } else {
        q.seq0 = v - a.n_groups;
        q.seq1 = q.seq0 + 1;
        q.key1 = clampi(a.context_lens ? a.context_lens[q.seq0] : 0, 0, cap);
        q.key0 = q.prefix = min(prefix_of(a, q.seq0), q.key1);
        q.new0 = clampi(a.cu_new[q.seq0], 0, a.n_new);
        q.n_new = clampi(a.cu_new[q.seq1], q.new0, a.n_new) - q.new0;
    }
    q.table = q.seq0;
    q.tok0 = clampi(a.cu_q[q.seq0], 0, a.n_q);
    q.rows = (clampi(a.cu_q[q.seq1], q.tok0, a.n_q) - q.tok0) * a.group_heads;
    q.narrow = q.rows <= kNarrowRows;
    const int kt = q.narrow ? kNarrowKeys : kWideKeys, rt = q.narrow ? kNarrowRows : kWideRows;
    q.row_tiles = (q.rows + rt - 1) / rt;
    q.ctx_tiles = (q.key1 - q.key0 + kt - 1) / kt;
    q.tiles = q.rows > 0 ? q.ctx_tiles + (q.n_new + kt - 1) / kt : 0;
    return q;
}

// Workgroup ranges: workgroup w owns the units that start at a cost in [floor(w U / W), floor((w + 1) U / W)).
DFX_D int64_t range_start(int w, int64_t total, int n_wg) { return w * total / n_wg; }
DFX_D int owner_of(int64_t cost, int64_t total, int n_wg) { return static_cast<int>(((cost + 1) * n_wg - 1) / total); }

// ---- one wave's 32 rows ------------------------------------------------------------------------
template <int HD>
struct Wave {
    using L = TileLayout<HD>;
    static constexpr int NSLAB = HD / 16, NDB = HD / 32;
    f32x16 o[NDB];
    bf16x8 q[NSLAB];
    float m, l;
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
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    }

    DFX_D void load_q(const uint16_t* row) {  // nullptr: a lane without a row
#pragma unroll
        for (int s = 0; s < NSLAB; ++s) {
            u32x4 w = {0, 0, 0, 0};
            if (row != nullptr) w = *reinterpret_cast<const u32x4*>(row + s * 16 + half * 8);
            q[s] = __builtin_bit_cast(bf16x8, w);
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

    // S^T = K Q^T, softmax, O^T += V^T P^T over KT keys in LDS.  `seen`: this lane's visible keys, looked at where !full.
    template <int KT>
    DFX_D void tile(uint32_t kt, uint32_t vt, float c, bool full, uint64_t seen) {
        constexpr int NT = KT / 32;
        typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
        typedef short short4v __attribute__((ext_vector_type(4)));
        typedef short short8v __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) short4v lds_short4v;
        f32x16 s[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
        for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const bf16x8 k = *(const lds_bf16x8*)static_cast<uintptr_t>(((kt + k_lane) ^ (sl * 32)) + t * 32 * L::ROWB);
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[sl], s[t], 0, 0, 0);
            }
        if (!full) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t bits = static_cast<uint32_t>(seen >> (32 * t)) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(bits & (1u << (8 * (i >> 2) + (i & 3))))) s[t][i] = -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
        top = half_max(top) * c;
        // The running maximum moves only where a tile's is more than 2^8 above it (or there is none yet): the
        // weights then stay below 2^8, far inside bf16 and fp32, and the accumulators are rarely rescaled.
        if (__builtin_amdgcn_ballot_w64(top > m + 8.0f)) {
            const float next = fmaxf(m, top);
            const float alpha = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        bf16x8 p[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float e[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], c, -base));
                l += e[i];
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{e[8 * x + 2 * i], e[8 * x + 2 * i + 1]}, bf16x2));
                p[t][x] = __builtin_bit_cast(bf16x8, w);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int d = 0; d < NDB; ++d) {
                    short4v r[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        r[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_short4v*)static_cast<uintptr_t>(((vt + v_lane) ^ (((d * 4) ^ L::swizzle(i * 8)) * 16)) +
                                                                 (t * 32 + x * 16 + i * 8) * L::ROWB));
                    const short8v v = __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), p[t][x], o[d], 0, 0, 0);
                }
    }
};

DFX_D void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- a workgroup's walk over its units ---------------------------------------------------------
template <int HD, int KV>
struct Split {
    using L = TileLayout<HD>;
    using W = Wave<HD>;
    static constexpr int NDB = HD / 32;
    static constexpr int kRowBytes = KV == kBf16 ? HD * 2 : KV == kMx8 ? HD : HD / 2;  // codes of a head row
    static constexpr int kChunks = kRowBytes / 16;                                     // 16-byte chunks of them
    static constexpr int kNewChunks = HD / 8;                                          // of a fresh (bf16) row
    static constexpr int kTileBytes = kWideKeys * L::ROWB;
    static constexpr int kLds = 4 * kTileBytes;  // wide: two buffers of K and V; narrow: K and V of 32 keys per wave
    static constexpr int kAccBytes = 32 * HD * 4;

    const SplitArgs& a;
    uint8_t* lds;
    float* ml;     // [4 waves][m, l][32]
    int tid, wave, lane;
    W w;
    // the item
    Seq sq;
    int kvh, row_tile;
    int lim_ctx, lim_new;      // this lane's row sees cached keys below lim_ctx and fresh rows below lim_new
    int64_t head_off;

    DFX_D Split(const SplitArgs& args, uint8_t* smem, float* ml_, int tid_)
        : a(args), lds(smem), ml(ml_), tid(tid_), wave(uniform(tid_ >> 6)), lane(tid_ & 63), w(tid_ & 63) {}

    // Cache slot byte offset of key position pos (this lane's), -1 where there is none.
    DFX_D int64_t row_of(int pos) const {
        if (pos >= sq.key1) return -1;
        const int p = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page_size;
        if (p >= a.max_pages) return -1;
        const int page = a.block_tables[sq.table * a.bt_stride + p];
        if (page < 0 || page >= a.n_pages) return -1;
        return page * a.c_sp + (pos - p * a.page_size) * a.c_st;
    }

    // Rows of a KT-key tile that one wave moves: all of them (narrow) or its quarter (wide).
    template <int KT, int ROWS>
    struct Stage {
        static constexpr int kPer = 64 / kChunks > ROWS ? ROWS : 64 / kChunks;        // rows per load of the wave
        static constexpr int kLoads = ROWS / kPer;
        u32x4 k[kLoads], v[kLoads];
        uint8_t ks[kLoads], vs[kLoads];
        uint64_t valid;  // keys of the tile that have a cache row
        bool fresh;
    };

    static DFX_D int64_t shuffle64(int64_t x, int from) {
        const int lo = __builtin_amdgcn_ds_bpermute(from * 4, static_cast<int>(x));
        const int hi = __builtin_amdgcn_ds_bpermute(from * 4, static_cast<int>(x >> 32));
        return static_cast<int64_t>(static_cast<uint32_t>(lo)) | (static_cast<int64_t>(hi) << 32);
    }

    // row: lane l's cache row of key l of the tile (row_of).  Issues the loads of the wave's rows [r0, r0 + ROWS).
    template <int KT, int ROWS>
    DFX_D void issue(Stage<KT, ROWS>& st, int64_t row, int r0) const {
        using S = Stage<KT, ROWS>;
        st.fresh = false;
        st.valid = __builtin_amdgcn_ballot_w64(row >= 0);
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
            const int r = i * S::kPer + lane / kChunks, ch = lane % kChunks;
            const int64_t at = shuffle64(row, r0 + (r < ROWS ? r : 0));
            st.k[i] = st.v[i] = u32x4{0, 0, 0, 0};
            st.ks[i] = st.vs[i] = 0;
            if (at >= 0 && r < ROWS) {
                const int64_t off = at + head_off + ch * 16;
                st.k[i] = *reinterpret_cast<const u32x4*>(a.k_cache + off);
                st.v[i] = *reinterpret_cast<const u32x4*>(a.v_cache + off);
                if constexpr (KV != kBf16) {
                    const int64_t so = off / (KV == kMx8 ? 32 : 16);
                    st.ks[i] = a.k_scales[so];
                    st.vs[i] = a.v_scales[so];
                }
            }
        }
    }

    // Registers -> LDS, widened.
    template <int KT, int ROWS>
    DFX_D void commit(const Stage<KT, ROWS>& st, uint8_t* kt, uint8_t* vt, int r0) const {
        using S = Stage<KT, ROWS>;
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
            const int r = i * S::kPer + lane / kChunks, ch = lane % kChunks;
            if (S::kPer * kChunks < 64 && r >= ROWS) continue;
            if constexpr (KV == kBf16) {
                const int off = L::chunk_offset(r0 + r, ch);
                *reinterpret_cast<u32x4*>(kt + off) = st.k[i];
                *reinterpret_cast<u32x4*>(vt + off) = st.v[i];
            } else {
                const float ks = mx_scale_operand(st.ks[i]), vs = mx_scale_operand(st.vs[i]);
                constexpr int N = KV == kMx8 ? 2 : 4;
#pragma unroll
                for (int x = 0; x < N; ++x) {
                    const int off = L::chunk_offset(r0 + r, ch * N + x);
                    if constexpr (KV == kMx8) {
                        *reinterpret_cast<u32x4*>(kt + off) = mx_widen8_e4m3(u32x2{st.k[i][2 * x], st.k[i][2 * x + 1]}, ks);
                        *reinterpret_cast<u32x4*>(vt + off) = mx_widen8_e4m3(u32x2{st.v[i][2 * x], st.v[i][2 * x + 1]}, vs);
                    } else {
                        *reinterpret_cast<u32x4*>(kt + off) = mx_widen8_e2m1(st.k[i][x], ks);
                        *reinterpret_cast<u32x4*>(vt + off) = mx_widen8_e2m1(st.v[i][x], vs);
                    }
                }
            }
        }
    }

    // Fresh rows [j0, j0 + KT) (bf16 operands): straight to LDS, there are few of them.
    template <int ROWS>
    DFX_D void fresh_rows(int j0, uint8_t* kt, uint8_t* vt, int r0) const {
        constexpr int kPer = 64 / kNewChunks;
#pragma unroll
        for (int i = 0; i < ROWS / kPer; ++i) {
            const int r = r0 + i * kPer + lane / kNewChunks, ch = lane % kNewChunks;
            u32x4 kk = {0, 0, 0, 0}, vv = {0, 0, 0, 0};
            if (j0 + r < sq.n_new) {
                const int64_t t = sq.new0 + j0 + r;
                kk = *reinterpret_cast<const u32x4*>(a.k_new + t * a.kn_st + kvh * a.kn_sh + ch * 8);
                vv = *reinterpret_cast<const u32x4*>(a.v_new + t * a.vn_st + kvh * a.vn_sh + ch * 8);
            }
            const int off = L::chunk_offset(r, ch);
            *reinterpret_cast<u32x4*>(kt + off) = kk;
            *reinterpret_cast<u32x4*>(vt + off) = vv;
        }
    }

    static DFX_D uint64_t below(int n) { return n <= 0 ? 0 : (n >= 64 ? ~0ull : (1ull << n) - 1); }

    template <int KT>
    DFX_D void compute(const uint8_t* kt, const uint8_t* vt, int t, uint64_t valid) {
        const bool fresh = t >= sq.ctx_tiles;
        const int base = fresh ? (t - sq.ctx_tiles) * KT : sq.key0 + t * KT;
        const int visible = (fresh ? lim_new : lim_ctx) - base;
        const uint64_t all = KT == 64 ? ~0ull : (1ull << 32) - 1;
        const bool full = (fresh || (valid & all) == all) && __builtin_amdgcn_ballot_w64(visible < KT) == 0;
        w.template tile<KT>(TileMathAddress(kt), TileMathAddress(vt), a.c, full, below(visible) & (fresh ? ~0ull : valid));
    }
    static DFX_D uint32_t TileMathAddress(const uint8_t* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)); }

    DFX_D int64_t lane_row(int t, int kt) const {  // row of key `lane` of context tile t, -1 for fresh tiles
        return t < sq.ctx_tiles && lane < kt ? row_of(sq.key0 + t * kt + lane) : -1;
    }

    DFX_D void start_item(int rows_from) {
        head_off = kvh * a.c_sh;
        const int row = rows_from + w.col;
        const bool live = row < sq.rows;
        const int t = live ? row / a.group_heads : 0, g = live ? row - t * a.group_heads : 0;
        const int64_t tok = sq.tok0 + t;
        w.load_q(live ? a.q + tok * a.q_st + (static_cast<int64_t>(kvh) * a.group_heads + g) * a.q_sh : nullptr);
        w.reset();
        lim_ctx = live ? sq.key1 : INT32_MAX;
        lim_new = !live ? INT32_MAX : a.block_causal ? min(sq.n_new, (t / a.dbs + 1) * a.dbs) : sq.n_new;
    }

    // A group's rows whose sequence's context ends inside the prefix (or before it) see less of it.
    DFX_D void limit_rows(int rows_from) {
        const int row = rows_from + w.col;
        if (row >= sq.rows) return;
        const int tok = sq.tok0 + row / a.group_heads;
        int lo = sq.seq0, hi = sq.seq1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu_q[mid] <= tok) lo = mid;
            else hi = mid;
        }
        lim_ctx = min(sq.key1, max(a.context_lens ? a.context_lens[lo] : 0, 0));
    }
    DFX_D bool uneven_group(bool is_group) {
        if (!is_group) return false;
        bool any = false;
        for (int s = sq.seq0 + tid; s < sq.seq1; s += kWgThreads) any |= (a.context_lens ? a.context_lens[s] : 0) < sq.key1;
        return __syncthreads_or(any);
    }

    DFX_D float* acc_slot(int64_t slot) const { return reinterpret_cast<float*>(a.workspace + a.slot_off + slot * kAccBytes); }
    DFX_D float* ml_slot(int64_t slot) const { return reinterpret_cast<float*>(a.workspace + a.ml_off) + slot * 64; }

    // d block `d` of a row block: a piece to its slot, or the finished rows to the output.
    DFX_D void put(f32x16 o, int d, float inv, int rows_from, int64_t slot, bool direct) {
        const int row = rows_from + w.col;
        if (row >= sq.rows) return;
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
    DFX_D void wide(int u0, int u1, bool is_group, int64_t slot, bool direct) {
        using S = Stage<kWideKeys, kWideKeys / kWgWaves>;
        constexpr int ROWS = kWideKeys / kWgWaves;
        const int rows_from = row_tile * kWideRows + wave * 32;
        const bool uneven = uneven_group(is_group);
        start_item(rows_from);
        if (uneven) limit_rows(rows_from);
        const int r0 = wave * ROWS;
        S st;
        uint64_t valid = 0;
        int64_t row = lane_row(u0, kWideKeys);
        issue(st, row, r0);
        row = u0 + 1 < u1 ? lane_row(u0 + 1, kWideKeys) : -1;
        for (int u = u0; u < u1; ++u) {
            uint8_t* kt = lds + ((u - u0) & 1) * 2 * kTileBytes;
            uint8_t* vt = kt + kTileBytes;
            if (u < sq.ctx_tiles) commit(st, kt, vt, r0);
            else fresh_rows<ROWS>((u - sq.ctx_tiles) * kWideKeys, kt, vt, r0);
            valid = st.valid;
            if (u + 1 < u1) {
                issue(st, row, r0);
                row = u + 2 < u1 ? lane_row(u + 2, kWideKeys) : -1;
            }
            lds_barrier();
            compute<kWideKeys>(kt, vt, u, valid);
        }
        if (rows_from < sq.rows) {
            const float l = W::half_sum(w.l);
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            const bool fits = slot + wave < a.n_slots;
            if (direct || fits) {
#pragma unroll
                for (int d = 0; d < NDB; ++d) put(w.o[d], d, inv, rows_from, slot + wave, direct);
                if (!direct) ml_slot(slot + wave)[lane] = w.half ? l : w.m;
            }
        }
        lds_barrier();  // (the next item's tiles)
    }

    // ---- narrow --------------------------------------------------------------------------------
    DFX_D void narrow(int u0, int u1, bool is_group, int64_t slot, bool direct) {
        using S = Stage<kNarrowKeys, kNarrowKeys>;
        uint8_t* kt = lds + wave * 2 * (kNarrowKeys * L::ROWB);
        uint8_t* vt = kt + kNarrowKeys * L::ROWB;
        const bool uneven = uneven_group(is_group);
        start_item(row_tile * kNarrowRows);
        if (uneven) limit_rows(row_tile * kNarrowRows);
        S st;
        const int first = u0 + wave;
        int64_t row = first < u1 ? lane_row(first, kNarrowKeys) : -1;
        if (first < u1) issue(st, row, 0);
        row = first + kWgWaves < u1 ? lane_row(first + kWgWaves, kNarrowKeys) : -1;
        for (int u = first; u < u1; u += kWgWaves) {
            if (u < sq.ctx_tiles) commit(st, kt, vt, 0);
            else fresh_rows<kNarrowKeys>((u - sq.ctx_tiles) * kNarrowKeys, kt, vt, 0);
            const uint64_t valid = st.valid;
            if (u + kWgWaves < u1) {
                issue(st, row, 0);
                row = u + 2 * kWgWaves < u1 ? lane_row(u + 2 * kWgWaves, kNarrowKeys) : -1;
            }
            asm volatile("" ::: "memory");
            compute<kNarrowKeys>(kt, vt, u, valid);
            asm volatile("" ::: "memory");
        }
        // merge the four waves' states: each leaves its accumulators in its own LDS, wave d takes d block d
        const float l = W::half_sum(w.l);
        ml[wave * 64 + lane] = w.half ? l : w.m;
        f32x4* mine = reinterpret_cast<f32x4*>(lds + wave * kAccBytes);
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                mine[(d * 4 + x) * 64 + lane] = f32x4{w.o[d][4 * x], w.o[d][4 * x + 1], w.o[d][4 * x + 2], w.o[d][4 * x + 3]};
        lds_barrier();
        float top = -INFINITY, sum = 0.0f, f[kWgWaves];
#pragma unroll
        for (int i = 0; i < kWgWaves; ++i) top = fmaxf(top, ml[i * 64 + w.col]);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int i = 0; i < kWgWaves; ++i) {
            f[i] = __builtin_amdgcn_exp2f(ml[i * 64 + w.col] - base);
            sum += f[i] * ml[i * 64 + 32 + w.col];
        }
        if (wave < NDB) {
            f32x16 o;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                f32x4 s = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < kWgWaves; ++i) {
                    const f32x4 p = reinterpret_cast<const f32x4*>(lds + i * kAccBytes)[(wave * 4 + x) * 64 + lane];
                    // (a wave without a visible key adds nothing, whatever 0 * p would be)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[j] += f[i] == 0.0f ? 0.0f : f[i] * p[j];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) o[4 * x + j] = s[j];
            }
            const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
            if (direct || slot < a.n_slots) {
                put(o, wave, inv, row_tile * kNarrowRows, slot, direct);
                if (!direct && wave == 0) ml_slot(slot)[lane] = w.half ? sum : top;
            }
        }
        lds_barrier();
    }
};

// Inclusive scan of three values over the workgroup; returns the totals through the references' last thread.
struct Sums {
    int64_t cost;
    int blocks, comb;
};
DFX_D Sums scan_up(Sums v, int by) {
    Sums r;
    const int from = (threadIdx.x & 63) - by;
    const int at = (from < 0 ? 0 : from) * 4;
    const int lo = __builtin_amdgcn_ds_bpermute(at, static_cast<int>(v.cost)), hi = __builtin_amdgcn_ds_bpermute(at, static_cast<int>(v.cost >> 32));
    r.cost = static_cast<int64_t>(static_cast<uint32_t>(lo)) | (static_cast<int64_t>(hi) << 32);
    r.blocks = __builtin_amdgcn_ds_bpermute(at, v.blocks);
    r.comb = __builtin_amdgcn_ds_bpermute(at, v.comb);
    if (from < 0) r = Sums{0, 0, 0};
    return r;
}

template <int HD, int KV>
__global__ void __launch_bounds__(kWgThreads, 2) split_attn_kernel(const SplitArgs a) {
    using T = Split<HD, KV>;
    __shared__ __attribute__((aligned(256))) uint8_t lds[T::kLds];
    __shared__ float ml[kWgWaves * 64];
    __shared__ Sums wave_sum[kWgWaves];
    __shared__ int first_v, first_blocks;
    __shared__ int64_t first_cost;
    const int tid = threadIdx.x;

    // the work list: each thread a run of virtual sequences, then a scan
    const int n = a.n_groups + a.n_seqs;
    const int per = (n + kWgThreads - 1) / kWgThreads;
    Sums mine = {0, 0, 0};
    for (int i = 0; i < per; ++i) {
        const int v = tid * per + i;
        if (v >= n) break;
        const Seq s = seq_of(a, v);
        const int items = a.h_kv * s.row_tiles;
        mine.cost += static_cast<int64_t>(items) * s.tiles * s.cost();
        mine.blocks += items * s.row_blocks();
        if (v >= a.n_groups) mine.comb += a.h_kv * ((s.rows + 31) / 32);
    }
    Sums upto = mine;
#pragma unroll
    for (int by = 1; by < 64; by *= 2) {
        const Sums o = scan_up(upto, by);
        upto.cost += o.cost;
        upto.blocks += o.blocks;
        upto.comb += o.comb;
    }
    if ((tid & 63) == 63) wave_sum[tid >> 6] = upto;
    __syncthreads();
    Sums total = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < kWgWaves; ++i) {
        if (i < (tid >> 6)) {
            upto.cost += wave_sum[i].cost;
            upto.blocks += wave_sum[i].blocks;
            upto.comb += wave_sum[i].comb;
        }
        total.cost += wave_sum[i].cost;
        total.blocks += wave_sum[i].blocks;
        total.comb += wave_sum[i].comb;
    }
    int n_wg = a.n_wg;
    if (total.cost / kMinCost < n_wg) n_wg = static_cast<int>(max(total.cost / kMinCost, static_cast<int64_t>(1)));
    // neighbouring ranges (the row tiles that read the same keys) on one XCD: workgroups go to the eight in turn
    const int per_xcd = (n_wg + 7) / 8;
    const int wg = static_cast<int>(blockIdx.x) / 8 < per_xcd ? static_cast<int>(blockIdx.x) % 8 * per_xcd + static_cast<int>(blockIdx.x) / 8 : n_wg;
    if (blockIdx.x == 0) {  // for the merge
        if (tid == 0) *reinterpret_cast<Header*>(a.workspace) = Header{total.cost, n_wg, total.comb};
        Sums at = {upto.cost - mine.cost, upto.blocks - mine.blocks, upto.comb - mine.comb};
        for (int i = 0; i < per; ++i) {
            const int v = tid * per + i;
            if (v >= n) break;
            const Seq s = seq_of(a, v);
            const int items = a.h_kv * s.row_tiles;
            reinterpret_cast<TabEntry*>(a.workspace + a.tab_off)[v] = TabEntry{at.cost, at.blocks, 0};
            if (v >= a.n_groups) reinterpret_cast<int*>(a.workspace + a.comb_off)[v - a.n_groups] = at.comb;
            at.cost += static_cast<int64_t>(items) * s.tiles * s.cost();
            at.blocks += items * s.row_blocks();
            if (v >= a.n_groups) at.comb += a.h_kv * ((s.rows + 31) / 32);
        }
    }
    if (wg >= n_wg || total.cost == 0) return;
    const int64_t c0 = range_start(wg, total.cost, n_wg), c1 = range_start(wg + 1, total.cost, n_wg);
    if (c0 >= c1) return;
    if (upto.cost > c0 && upto.cost - mine.cost <= c0) {  // this thread's run holds the first unit
        int64_t cost = upto.cost - mine.cost;
        int blocks = upto.blocks - mine.blocks;
        for (int i = 0; i < per; ++i) {
            const int v = tid * per + i;
            const Seq s = seq_of(a, v);
            const int items = a.h_kv * s.row_tiles;
            const int64_t here = static_cast<int64_t>(items) * s.tiles * s.cost();
            if (cost + here > c0) {
                first_v = v;
                first_cost = cost;
                first_blocks = blocks;
                break;
            }
            cost += here;
            blocks += items * s.row_blocks();
        }
    }
    __syncthreads();
    int64_t cost = first_cost;
    int blocks = first_blocks;
    T t(a, lds, ml, tid);
    for (int v = uniform(first_v); v < n && cost < c1; ++v) {
        t.sq = seq_of(a, v);
        const Seq& s = t.sq;
        const int items = a.h_kv * s.row_tiles, unit = s.cost();
        const int64_t item_cost = static_cast<int64_t>(s.tiles) * unit;
        if (item_cost > 0) {
            int j = cost < c0 ? static_cast<int>((c0 - cost) / item_cost) : 0;
            for (; j < items; ++j) {
                const int64_t from = cost + j * item_cost;
                if (from >= c1) break;
                const int u0 = from >= c0 ? 0 : static_cast<int>((c0 - from + unit - 1) / unit);
                const int u1 = static_cast<int>(min(static_cast<int64_t>(s.tiles), (c1 - from + unit - 1) / unit));
                if (u0 >= u1) continue;
                t.kvh = j / s.row_tiles;
                t.row_tile = j - t.kvh * s.row_tiles;
                const bool is_group = v < a.n_groups;
                const bool direct = !is_group && s.prefix == 0 && u0 == 0 && u1 == s.tiles;
                const int64_t slot = static_cast<int64_t>(wg) * (kWideRows / 32) + blocks + j * s.row_blocks();
                if (s.narrow) t.narrow(u0, u1, is_group, slot, direct);
                else t.wide(u0, u1, is_group, slot, direct);
            }
        }
        cost += items * item_cost;
        blocks += items * s.row_blocks();
    }
}

// ---- merge -------------------------------------------------------------------------------------
// One workgroup per (sequence, KV head, 32 rows); wave d merges d block d (head_dim 64: two waves per d block, every
// second piece each).
template <int HD>
__global__ void __launch_bounds__(kWgThreads) split_merge_kernel(const SplitArgs a) {
    constexpr int NDB = HD / 32, kShare = kWgWaves / NDB;
    constexpr int kAccBytes = 32 * HD * 4;
    __shared__ int found;
    __shared__ float part[kWgWaves][18][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, half = lane >> 5;
    const Header h = *reinterpret_cast<const Header*>(a.workspace);
    const int x = blockIdx.x;
    if (x >= h.n_comb) return;
    const int* comb = reinterpret_cast<const int*>(a.workspace + a.comb_off);
    for (int s = tid; s < a.n_seqs; s += kWgThreads) {
        const int next = s + 1 < a.n_seqs ? comb[s + 1] : h.n_comb;
        if (comb[s] <= x && x < next) found = s;
    }
    __syncthreads();
    const int s = uniform(found), v = a.n_groups + s;
    const Seq q = seq_of(a, v);
    if (q.key1 == 0 && q.n_new == 0) return;  // no key at all: the rows stay as they are
    const int rbs = (q.rows + 31) / 32;
    const int local = x - comb[s], kvh = local / rbs, rb = local - kvh * rbs;
    const TabEntry* tab = reinterpret_cast<const TabEntry*>(a.workspace + a.tab_off);
    const int row = rb * 32 + col;
    const bool live = row < q.rows;

    // the pieces of this lane's row: own item, then the group's
    int w0[2] = {0, 0}, n[2] = {0, 0}, at_col[2] = {col, 0};
    int64_t slot0[2] = {0, 0};
    if (q.tiles > 0) {
        const int t = q.narrow ? rb : rb / 4;
        const int64_t j = static_cast<int64_t>(kvh) * q.row_tiles + t, unit = q.cost();
        const int64_t from = tab[v].cost + j * q.tiles * unit;
        w0[0] = owner_of(from, h.total, h.n_wg);
        n[0] = owner_of(from + (q.tiles - 1) * unit, h.total, h.n_wg) - w0[0] + 1;
        slot0[0] = tab[v].blocks + j * q.row_blocks() + (q.narrow ? 0 : rb & 3);
        if (q.prefix == 0 && n[0] == 1) return;  // written by its only workgroup
    }
    if (q.prefix > 0) {
        int lo = 0, hi = a.n_groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.group_cu[mid] <= s) lo = mid;
            else hi = mid;
        }
        const Seq g = seq_of(a, lo);
        if (g.tiles > 0) {
            const int grow = (q.tok0 - g.tok0) * a.group_heads + row;
            const int rt = g.narrow ? kNarrowRows : kWideRows, t = grow / rt;
            const int64_t j = static_cast<int64_t>(kvh) * g.row_tiles + t, unit = g.cost();
            const int64_t from = tab[lo].cost + j * g.tiles * unit;
            w0[1] = owner_of(from, h.total, h.n_wg);
            n[1] = live ? owner_of(from + (g.tiles - 1) * unit, h.total, h.n_wg) - w0[1] + 1 : 0;
            slot0[1] = tab[lo].blocks + j * g.row_blocks() + (grow - t * rt) / 32;
            at_col[1] = grow & 31;
        }
    }
    const int d = wave % NDB, share = wave / NDB;
    float m = -INFINITY, l = 0.0f;
    f32x4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
        const int c = at_col[kind];
        for (int i = share; __builtin_amdgcn_ballot_w64(i < n[kind]) != 0; i += kShare) {
            const int64_t slot = slot0[kind] + static_cast<int64_t>(w0[kind] + i) * (kWideRows / 32);
            if (!live || i >= n[kind] || slot >= a.n_slots) continue;
            const float* ml = reinterpret_cast<const float*>(a.workspace + a.ml_off) + slot * 64;
            const f32x4* acc = reinterpret_cast<const f32x4*>(a.workspace + a.slot_off + slot * kAccBytes);
            const float pm = ml[c], pl = ml[32 + c];
            f32x4 po[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) po[y] = acc[(d * 4 + y) * 64 + half * 32 + c];
            if (pm == -INFINITY && pl == 0.0f) continue;  // no visible key in the piece
            const float next = fmaxf(m, pm);
            const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - next), add = __builtin_amdgcn_exp2f(pm - next);
            m = next;
            l = l * keep + pl * add;
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int z = 0; z < 4; ++z) o[y][z] = o[y][z] * keep + po[y][z] * add;
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
        const int other = wave + NDB;
        const float pm = part[other][0][lane], pl = part[other][1][lane];
        const float next = fmaxf(m, pm), base = next == -INFINITY ? 0.0f : next;
        const float keep = __builtin_amdgcn_exp2f(m - base), add = __builtin_amdgcn_exp2f(pm - base);
        l = l * keep + pl * add;
#pragma unroll
        for (int y = 0; y < 16; ++y) o[y >> 2][y & 3] = o[y >> 2][y & 3] * keep + part[other][2 + y][lane] * add;
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

// Sizes of the launch and of its workspace; a status.
int lay_out(const dfx_split_attn_params* p, SplitArgs& a, int64_t& comb_blocks, int64_t& bytes) {
    if (!p || p->num_seqs < 0 || p->num_groups < 0 || p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->num_q_tokens < 0 ||
        p->num_new_tokens < 0 || p->max_workgroups < 0)
        return DFX_ERR_INVALID_ARG;
    if (p->num_q_heads % p->num_kv_heads != 0) return DFX_ERR_INVALID_ARG;
    if (p->head_dim != 64 && p->head_dim != 128) return DFX_ERR_UNSUPPORTED;
    if (p->num_seqs > 65535 || p->num_groups > p->num_seqs + 1 || p->num_q_tokens > INT32_MAX / p->num_q_heads ||
        p->num_new_tokens > INT32_MAX || p->max_workgroups > 65535)
        return DFX_ERR_UNSUPPORTED;
    int n_wg = p->max_workgroups;
    if (n_wg == 0) {
        const int cus = compute_units();
        if (cus < 0) return DFX_ERR_LAUNCH;
        n_wg = 2 * cus;
    }
    a.n_wg = n_wg;
    a.n_seqs = p->num_seqs;
    a.n_groups = p->num_groups;
    a.h_kv = p->num_kv_heads;
    a.group_heads = p->num_q_heads / p->num_kv_heads;
    const int64_t rows32 = (p->num_q_tokens * a.group_heads + 31) / 32;
    comb_blocks = a.h_kv * (rows32 + p->num_seqs);
    // (an item of R rows takes at most R / 32 + 4 blocks)
    const int64_t blocks = a.h_kv * ((p->num_groups > 0 ? 2 : 1) * rows32 + 4 * (static_cast<int64_t>(p->num_seqs) + p->num_groups));
    a.n_slots = static_cast<int64_t>(n_wg) * (kWideRows / 32) + blocks;
    if (comb_blocks > UINT32_MAX / kWgThreads || blocks > INT32_MAX) return DFX_ERR_UNSUPPORTED;
    a.tab_off = 256;
    a.comb_off = a.tab_off + round_up((static_cast<int64_t>(p->num_seqs) + p->num_groups) * static_cast<int64_t>(sizeof(TabEntry)), 256);
    a.ml_off = a.comb_off + round_up(static_cast<int64_t>(p->num_seqs) * 4, 256);
    a.slot_off = a.ml_off + a.n_slots * 256;
    bytes = a.slot_off + a.n_slots * 32 * p->head_dim * 4;
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
    if (p->k_cache) {
        if (!p->v_cache || !p->block_tables || !p->context_lens || p->page_size <= 0 || p->n_pages < 0 || p->max_pages_per_seq < 0 ||
            p->block_table_stride < 0)
            return DFX_ERR_INVALID_ARG;
        if (mx != (p->k_scales != nullptr) || mx != (p->v_scales != nullptr)) return DFX_ERR_INVALID_ARG;
        if (p->n_pages > INT32_MAX) return DFX_ERR_UNSUPPORTED;
        const int64_t row = mx ? mx_row_bytes(p->kv_dtype == DFX_KV_MX_E2M1, p->head_dim) : 0;
        if (mx) {
            a.c_sh = row;
            a.c_st = row * p->num_kv_heads;
            a.c_sp = a.c_st * p->page_size;
        } else {
            if (p->cache_stride_page % 8 || p->cache_stride_token % 8 || p->cache_stride_head % 8 || p->cache_stride_page < 0 ||
                p->cache_stride_token < 0 || p->cache_stride_head < 0)
                return DFX_ERR_INVALID_ARG;
            a.c_sp = p->cache_stride_page * 2;
            a.c_st = p->cache_stride_token * 2;
            a.c_sh = p->cache_stride_head * 2;
        }
        a.block_tables = p->block_tables;
        a.context_lens = p->context_lens;
        a.bt_stride = p->block_table_stride;
        a.n_pages = static_cast<int>(p->n_pages);
        a.max_pages = p->max_pages_per_seq;
        a.page_size = p->page_size;
        a.page_shift = (p->page_size & (p->page_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(p->page_size)) : -1;
    } else {
        a.page_size = 1;
    }
    if (!p->workspace || p->workspace_bytes < bytes) return DFX_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(p->workspace) % 256) return DFX_ERR_INVALID_ARG;
    a.q = static_cast<const uint16_t*>(p->q);
    a.k_new = static_cast<const uint16_t*>(p->k_new);
    a.v_new = static_cast<const uint16_t*>(p->v_new);
    a.out = static_cast<uint16_t*>(p->out);
    a.k_cache = static_cast<const uint8_t*>(p->k_cache);
    a.v_cache = static_cast<const uint8_t*>(p->v_cache);
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
    const dim3 grid(static_cast<unsigned>(a.n_wg)), block(kWgThreads), merge(static_cast<unsigned>(comb));
    const int kv = !a.k_cache || !mx ? kBf16 : p->kv_dtype == DFX_KV_MX_E4M3 ? kMx8 : kMx4;
#define DFX_SPLIT(HD_)                                                                                      \
    do {                                                                                                    \
        auto kern = kv == kBf16 ? split_attn_kernel<HD_, kBf16>                                             \
                                : kv == kMx8 ? split_attn_kernel<HD_, kMx8> : split_attn_kernel<HD_, kMx4>; \
        hipLaunchKernelGGL(kern, grid, block, 0, st, a);                                                    \
        hipLaunchKernelGGL((split_merge_kernel<HD_>), merge, block, 0, st, a);                              \
    } while (0)
    if (p->head_dim == 128) DFX_SPLIT(128);
    else DFX_SPLIT(64);
#undef DFX_SPLIT
    return launch_status();
}
