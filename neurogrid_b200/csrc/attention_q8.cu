// Tensor-core attention over a paged cache in 8 bits (ng_q8.cuh), specialised on the head size (compile with -DNG_HEAD_DIM=<multiple of
// 16, 16..256>): single tokens, split over the context, and portions.
//
// With codes c and d, block scales s and t, and one row of q:  x_j = scale (q . c_j) s_j - slope (pos - j),
//     out = sum_j e^(x_j) t_j d_j / sum_j e^(x_j).
// The codes go into the MMAs as they are (float16, exact); q goes in as float16 after a division by a power of two of its own
// (more of its bits than bfloat16 has survive: values 2^-14 and less of the row's largest lose some of theirs).  s_j multiplies the 32-bit
// score.  t_j goes into the exponent: with z_j = x_j log2(e) + log2(t_j) and the reference point m near max z_j, the weights
// w_j = 2^(z_j - m) are what meets the codes d_j, in float16 (half a step 2^-12 of the weight, smallest step 2^-24 of the
// largest), and the denominator is sum_j w_j / t_j in 32 bits: t_j is a power of two, both forms are exact.  So a block
// whose values are small has small weights, not small values, and the sum over the codes never leaves float16's range.  Where scales lie so far
// apart (Q8_LOW) that a w_j may be lost which counts in the denominator, the denominator takes 2^(x_j log2(e) - m) by an exponential of
// its own, and its sums are moved in two steps where one factor would be lost.
// Entries whose context is below zero or behind the table's last place are passed over, their rows left as they were.  Keys whose page is not there
// (below zero, or beyond the pool) are hidden from every row.
#include "ng_q8_attention.cuh"

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// ===================================================================================== single tokens
// A segment is an entry's keys for up to 8 NT query heads of one KV head.  The block's four warps take groups of GROUP keys in turn, each on
// its own (no barrier until the end of a piece).  Keys are the rows of the first product's tiles and dimensions those of the second's,
// S^T = K Q^T and O^T = V^T P^T, so that up to eight heads fill a tile's columns: half the products, exponentials and
// accumulators of heads as rows (16 of them, of which eight stay empty).  The contraction index of the first and the row index of the second are
// permuted so that a lane reads contiguous bytes.  K and V come from memory into the registers they are used from, the next group's requested
// before this group is computed and the page numbers a group earlier still; nothing passes through shared memory but the four warps' results.
//
// A lane's words of V hold one key's codes each; a byte permutation puts a pair of keys beside each other, as the MMA wants them, and a movmatrix
// turns a tile of weights from keys x heads to heads x keys.
//
// Who does what: with one run, a block has a segment.  With more, the launch has as many blocks as the GPU holds at once, in teams of a block for
// each segment of an entry, and every team finds, from the entries' lengths on the device, its equal share of the turns of all entries
// laid end to end: pieces of one entry or several.  A piece that is a whole segment writes its output rows; others write records for the
// merge, the piece's number within the segment as the run's.  So batches of unequal lengths, and segments a little more than the blocks, fill
// the GPU evenly.
//
// Bound by the codes' bytes where there are many (2 requests behind 131,072 tokens, 32 / 8 heads of 128: 87.5 us, 6.1 TB/s = 0.94 of a plain copy's rate) and else by
// the chain of a group: page numbers -> codes -> products -> maximum -> weights -> products, three blocks an SM wide (64 requests of
// up to 4,096 tokens, 32 / 8 heads of 64, integers: 39.5 us, 4.3 TB/s; the loads alone take 33, the arithmetic alone 34).  8 requests behind
// 2,100 tokens 10.0 us, 1 behind 300 4.2 us.  Codes through a ring in shared memory (cp.async, 2 to 4 stages) took 43 to 48 us for the 64 requests
// (more work for the load and store unit), groups of 16 keys or of 64 were slower with heads of 64, conversions cost nothing that could be seen.
#define DC_WARPS 4
#define DC_THREADS (DC_WARPS * 32)
constexpr int W = HD % 64 == 0 ? 16 : HD % 32 == 0 ? 8 : 4;        // bytes of a key that a lane takes at once (of a value row: half of it)
constexpr int NC = HD / (4 * W);                                    // such pieces a row has for it
constexpr int VW = (W / 2 + 3) / 4;                                 // words that hold a value row's piece
constexpr int SUB = HD <= 128 ? 2 : 1;                              // 16-key tiles a group has
constexpr int GROUP = 16 * SUB;
constexpr int DC_NT_MAX = HD <= 64 ? 2 : 1;                         // 8 heads wide; more heads are blocks of their own

// GRAN (8 or 16): keys that certainly lie in one page and one block; a unit is so many
template <int GRAN>
struct DcGroup {
    static constexpr int UNITS = 16 / GRAN;
    uint32_t k[SUB][2][NC * W / 4];          // keys g and 8 + g of the tile
    uint32_t v[SUB][4][NC * VW];             // keys 2t, 2t+1, 8+2t, 8+2t+1
    float ks[SUB][UNITS], vs[SUB][UNITS];
    uint32_t missing;                        // a bit for each unit whose page is not there
};
template <int GRAN>
struct DcPages { int id[SUB][16 / GRAN]; };
// where a lane's pieces of a page's keys and values begin (the pointers of page 0), and what a page is long
struct DcBase {
    const unsigned char *k, *v;
    const float *ks, *vs;
    int page_bytes, page_scales, slot_mask, bl_log2;
};

template <int GRAN>
__device__ __forceinline__ void dc_pages(DcPages<GRAN>& p, const Cache& c, const int* trow, int key0, int k_end) {
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int u = 0; u < 16 / GRAN; ++u) {
            const int key = key0 + 16 * s + GRAN * u, i = key >> c.ps_log2;
            p.id[s][u] = key < k_end && i < c.table_stride ? trow[i] : -1;
        }
}
// Keys key0 .. key0 + GROUP - 1 of the block's run.  Of a page that is not there, or a unit behind the run, page 0 is read: the group's keys
// are then looked at one by one.
template <int GRAN>
__device__ __forceinline__ void dc_load(DcGroup<GRAN>& r, const DcBase& b, const DcPages<GRAN>& p, int key0, int num_pages) {
    r.missing = 0;
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int u = 0; u < 16 / GRAN; ++u) {
            int id = p.id[s][u];
            if ((unsigned)id >= (unsigned)num_pages) {
                id = 0;
                r.missing |= 1u << (s * (16 / GRAN) + u);
            }
            const int slot = (key0 + 16 * s + GRAN * u) & b.slot_mask;
            const long long at = (long long)id * b.page_bytes + slot * HD;
            const long long sc = (long long)id * b.page_scales + (slot >> b.bl_log2);
            r.ks[s][u] = b.ks[sc];
            r.vs[s][u] = b.vs[sc];
#pragma unroll
            for (int h = 0; h < GRAN / 8; ++h) {
                const int half = GRAN == 8 ? u : h;
#pragma unroll
                for (int n = 0; n < NC; ++n) ld_codes<W>(&r.k[s][half][n * (W / 4)], b.k + at + h * 8 * HD + n * 4 * W);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int n = 0; n < NC; ++n) ld_codes<W / 2>(&r.v[s][2 * half + j][n * VW], b.v + at + (h * 8 + j) * HD + n * 4 * W);
            }
        }
}

// Of the heads 2t and 2t+1 (and, for the second tile of heads, 8 + those): accumulators, reference point, sum.
template <int NT>
struct DcState {
    float o[NT][HD / 16][4], m[NT][2], l[NT][2];
    uint32_t seen;                           // a bit for each (tile of heads, of the lane's two): a finite score has been met; the highest: Q8_HIGH
};
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// One group into the warp's state.  f: what the raw products of the lane's heads are multiplied by (base 2).
template <int KIND, int NT, int GRAN>
__device__ __forceinline__ void dc_compute(DcState<NT>& st, DcGroup<GRAN>& r, const uint32_t (&qb)[NT][HD / 16][2], int key0, int key_lo,
                                           int k_end, int pos, const float (&f)[NT][2], const float (&slope)[NT][2], bool biased) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    constexpr int UNITS = 16 / GRAN;
    float sc[NT][SUB][4];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][s][0] = sc[n][s][1] = sc[n][s][2] = sc[n][s][3] = 0.f;
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            uint32_t a[4];
            q8_to_half<KIND>(r.k[s][0][i], a[0], a[2]);
            q8_to_half<KIND>(r.k[s][1][i], a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(sc[n][s], a, qb[n][i][0], qb[n][i][1]);
        }
    const bool whole = key0 >= key_lo && key0 + GROUP <= k_end && r.missing == 0;
    if (!whole)                                                      // scales of units that no key is seen of may be NaN
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const int key = key0 + 16 * s + GRAN * u;
                if (key >= k_end || key + GRAN <= key_lo || (r.missing >> (s * UNITS + u) & 1)) r.ks[s][u] = r.vs[s][u] = 1.f;
            }
    bool wide = false;                                               // (Q8_LOW)
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int u = 0; u < UNITS; ++u) wide = wide || r.vs[s][u] < q8_pow2(Q8_LOW);
    // z less the reference point as it stands: what 2^ is taken of, unless the point has to move
    float mx[NT][2];
    bool up = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mx[n][0] = mx[n][1] = -INFINITY;
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const float lg = q8_log2(r.vs[s][u]);
#pragma unroll
                for (int j = 0; j < 4 / UNITS; ++j) {                // of a unit: [half of the tile,] head
                    const int c = UNITS == 1 ? j : 2 * u + j;
                    sc[n][s][c] = fmaf(sc[n][s][c], f[n][j & 1] * r.ks[s][u], lg - st.m[n][j & 1]);
                }
            }
        if (biased || !whole)
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + 16 * s + 8 * (j >> 1) + g;
                    const bool seen = whole || (key >= key_lo && key < k_end && !(r.missing >> (s * UNITS + (j >> 1) * (UNITS - 1)) & 1));
                    sc[n][s][j] = seen ? fmaf(-slope[n][j & 1], (float)(pos - key), sc[n][s][j]) : -INFINITY;
                }
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) mx[n][j & 1] = fmaxf(mx[n][j & 1], sc[n][s][j]);
        up |= fmaxf(mx[n][0], mx[n][1]) > 8.f || (st.seen >> 2 * n & 3) != 3;
    }
    // the reference point follows the maximum lazily: weights may reach 2^8 before the sums are rescaled.  It starts at 0 and moves to a head's
    // first maximum, up or down, with sums that are zero.  Each head has its own bit for that: one whose scores are all NaN never gets it.
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
                if (r.vs[s][u] > q8_pow2(Q8_HIGH)) st.seen |= 1u << 31;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = mx[n][j];                                  // (the same in every lane that has the head: so is the bit)
#pragma unroll
                for (int o = 4; o <= 16; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                const bool first = !(st.seen >> (2 * n + j) & 1);
                const float by = x == -INFINITY ? 0.f : first ? x : fmaxf(x, 0.f), c = first ? 1.f : q8_ex2(-by);
                st.m[n][j] += by;
                if (!first) st.l[n][j] = q8_add_scaled(st.l[n][j], -by, 0.f);
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) { st.o[n][i][j] *= c; st.o[n][i][2 + j] *= c; }
                if (x != -INFINITY) st.seen |= 1u << (2 * n + j);
#pragma unroll
                for (int s = 0; s < SUB; ++s) { sc[n][s][j] -= by; sc[n][s][2 + j] -= by; }
            }
        }
    }
    if (wide || st.seen >> 31)                                       // in place of what is added below
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float vs = r.vs[s][UNITS == 1 ? 0 : j >> 1];
                    st.l[n][j & 1] += q8_ex2(sc[n][s][j] - q8_log2(vs)) - q8_ex2(sc[n][s][j]) * q8_recip(vs);
                }
    uint32_t pb[NT][SUB][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            float p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = q8_ex2(sc[n][s][j]);
            if constexpr (UNITS == 1) {
                const float inv = q8_recip(r.vs[s][0]);
                st.l[n][0] = fmaf(p[0] + p[2], inv, st.l[n][0]);
                st.l[n][1] = fmaf(p[1] + p[3], inv, st.l[n][1]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) st.l[n][j & 1] = fmaf(p[j], q8_recip(r.vs[s][j >> 1]), st.l[n][j & 1]);
            }
            pb[n][s][0] = movmatrix(pack_f16(p[0], p[1]));
            pb[n][s][1] = movmatrix(pack_f16(p[2], p[3]));
        }
    }
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
        if (!whole)                                                  // a key that no row sees has a weight of 0, but its codes may be NaN
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = key0 + 16 * s + 8 * (j >> 1) + 2 * t + (j & 1);
                if (key < key_lo || key >= k_end || (r.missing >> (s * UNITS + (j >> 1) * (UNITS - 1)) & 1))
#pragma unroll
                    for (int i = 0; i < NC * VW; ++i) r.v[s][j][i] = 0u;
            }
#pragma unroll
        for (int i = 0; i < NC * VW; ++i)                            // a word: four dimensions (two where W is 4), two tiles (one)
#pragma unroll
            for (int d = 0; d < (W >= 8 ? 2 : 1); ++d) {
                uint32_t a[4];
                q8_to_half<KIND>(__byte_perm(r.v[s][0][i], r.v[s][1][i], d ? 0x7362 : 0x5140), a[0], a[1]);
                q8_to_half<KIND>(__byte_perm(r.v[s][2][i], r.v[s][3][i], d ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(st.o[n][W >= 8 ? 2 * i + d : i], a, pb[n][s][0], pb[n][s][1]);
            }
    }
}
// the dimension that rows g (upper 0) and g + 8 (upper 1) of tile i of O^T are
__device__ __forceinline__ int dc_dim(int i, int g, int upper) {
    constexpr int PER = W / 2;                                       // dimensions a lane group has of a piece
    return (2 * i / PER) * 8 * PER + g * PER + 2 * i % PER + upper;
}

struct DcArgs {
    Cache c;
    const bf16* q;
    const int *cu_q, *ctx_before;
    bf16* out;
    float* scratch;
    const float* slopes;
    int n_rows, n_entries, nH, chunks, window, n_splits;
    float scale;
};
constexpr int TURN = DC_WARPS * GROUP;                               // keys of a turn of the four warps
// turns of an entry's segments (0: not a single token, or a row that the buffers, or a position that the table, do not hold)
__device__ __forceinline__ int dc_turns(const DcArgs& a, int e) {
    const int row = a.cu_q[e], pos = a.ctx_before[e];
    if (a.cu_q[e + 1] - row != 1 || row < 0 || row >= a.n_rows || pos < 0 || pos > a.c.last_key) return 0;
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) & ~(GROUP - 1) : 0;
    return (pos - lo) / TURN + 1;
}

// A team is a block for each segment of an entry; its blocks have the same share of the keys, so that the heads of a page, which lie side by side in
// memory, are read at about the same time.  The team's share: turns [first, last) of all entries laid end to end, of which entry e's begin at
// `before`.  Every warp finds it for itself, 32 entries at a time.  Few entries: they count as whole multiples of the share, so that no team has
// pieces of two.
struct DcShare { int first, last, each, before, e; bool even; };
__device__ __forceinline__ int dc_length(const DcShare& sh, int turns) { return sh.even ? (turns + sh.each - 1) / sh.each * sh.each : turns; }
__device__ __forceinline__ DcShare dc_share(const DcArgs& a, int team, int teams) {
    const int lane = threadIdx.x & 31;
    int total = 0, most = 0, live = 0;
    for (int e0 = 0; e0 < a.n_entries; e0 += 32) {
        const int n = e0 + lane < a.n_entries ? dc_turns(a, e0 + lane) : 0;
        total += __reduce_add_sync(0xffffffffu, n);
        most = max(most, __reduce_max_sync(0xffffffffu, n));
        live += __popc(__ballot_sync(0xffffffffu, n > 0));
    }
    DcShare sh;
    sh.even = 4 * live <= teams;
    // none so small that an entry has more pieces than there are records for
    sh.each = max(sh.even ? (total + teams - live - 1) / max(1, teams - live) : (total + teams - 1) / teams,
                  (most + a.n_splits - 2) / (a.n_splits - 1));
    sh.each = max(sh.each, 1);
    sh.first = sh.last = sh.before = sh.e = 0;
    const long long want = (long long)sh.each * team;
    int before = 0;
    for (int e0 = 0; e0 < a.n_entries; e0 += 32) {
        const int n = e0 + lane < a.n_entries ? dc_length(sh, dc_turns(a, e0 + lane)) : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const uint32_t in = __ballot_sync(0xffffffffu, want < before + upto);
        if (in) {
            const int l = __ffs(in) - 1;
            sh.before = before + __shfl_sync(0xffffffffu, upto - n, l);
            sh.e = e0 + l;
            sh.first = (int)want;
            sh.last = sh.first + sh.each;                            // (the caller stops behind the last entry)
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return sh;
}

template <int KIND, int NT, int GRAN>
__device__ __forceinline__ void dc_piece(const DcArgs& a, float* red_s, int e, int segment, int turn0, int turn1, int run, int runs) {
    const int row = a.cu_q[e], pos = a.ctx_before[e], kvh = segment / a.chunks;
    const int G = a.nH / a.c.nKV, h0 = (segment - kvh * a.chunks) * 8 * NT, heads = min(8 * NT, G - h0);
    const int head0 = kvh * G + h0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int key_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int k_begin = (key_lo & ~(GROUP - 1)) + turn0 * TURN, k_end = min(pos + 1, k_begin + (turn1 - turn0) * TURN);
    const int* trow = a.c.table + (size_t)e * a.c.table_stride;
    constexpr int STEP = TURN;

    DcGroup<GRAN> cur, nxt;
    DcPages<GRAN> pages;
    DcBase base;
    base.page_scales = a.c.nKV << (a.c.ps_log2 - a.c.bl_log2);
    base.page_bytes = (a.c.nKV << a.c.ps_log2) * HD;
    base.k = a.c.k + (kvh << a.c.ps_log2) * HD + g * HD + t * W;
    base.v = a.c.v + (kvh << a.c.ps_log2) * HD + 2 * t * HD + g * (W / 2);
    base.ks = a.c.ks + (kvh << (a.c.ps_log2 - a.c.bl_log2));
    base.vs = a.c.vs + (kvh << (a.c.ps_log2 - a.c.bl_log2));
    base.slot_mask = (1 << a.c.ps_log2) - 1;
    base.bl_log2 = a.c.bl_log2;
    int key0 = k_begin + warp * GROUP;
    if (key0 < k_end) {
        dc_pages(pages, a.c, trow, key0, k_end);
        dc_load(cur, base, pages, key0, a.c.num_pages);
        dc_pages(pages, a.c, trow, key0 + STEP, k_end);
    }
    // columns of the MMA tiles: the block's heads (beyond them: zeros), each divided by a power of two
    uint32_t qb[NT][HD / 16][2];
    float f[NT][2], slope[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int h = 8 * n + g;
        const bf16* q = ng_after_wait(a.q) + ((size_t)row * a.nH + head0 + h) * HD;
        uint2 w[HD / 16];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            const int d = (i / (W / 4)) * 4 * W + t * W + (i % (W / 4)) * 4;
            w[i] = h < heads ? *reinterpret_cast<const uint2*>(q + d) : make_uint2(0u, 0u);
            const uint32_t x[4] = {w[i].x << 16, w[i].x & 0xffff0000u, w[i].y << 16, w[i].y & 0xffff0000u};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = fabsf(__uint_as_float(x[j]));
                top = v < INFINITY ? fmaxf(top, v) : top;
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = q_exponent(top);
        const float div = pow2_any(-ex), mul = a.scale * LOG2E * pow2_any(ex);
        const float sl = a.slopes && h < heads ? a.slopes[head0 + h] * LOG2E : 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            qb[n][i][0] = pack_f16(__uint_as_float(w[i].x << 16) * div, __uint_as_float(w[i].x & 0xffff0000u) * div);
            qb[n][i][1] = pack_f16(__uint_as_float(w[i].y << 16) * div, __uint_as_float(w[i].y & 0xffff0000u) * div);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f[n][j] = __shfl_sync(0xffffffffu, mul, (2 * t + j) * 4);
            slope[n][j] = __shfl_sync(0xffffffffu, sl, (2 * t + j) * 4);
        }
    }
    DcState<NT> st;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) st.o[n][i][0] = st.o[n][i][1] = st.o[n][i][2] = st.o[n][i][3] = 0.f;
        st.m[n][0] = st.m[n][1] = st.l[n][0] = st.l[n][1] = 0.f;
    }
    st.seen = 0;
    const bool biased = a.slopes != nullptr;
    if constexpr (HD <= 128) {
        for (; key0 < k_end; key0 += 2 * STEP) {
            if (key0 + STEP < k_end) {
                dc_load(nxt, base, pages, key0 + STEP, a.c.num_pages);
                dc_pages(pages, a.c, trow, key0 + 2 * STEP, k_end);
            }
            dc_compute<KIND, NT, GRAN>(st, cur, qb, key0, key_lo, k_end, pos, f, slope, biased);
            if (key0 + STEP >= k_end) break;
            if (key0 + 2 * STEP < k_end) {
                dc_load(cur, base, pages, key0 + 2 * STEP, a.c.num_pages);
                dc_pages(pages, a.c, trow, key0 + 3 * STEP, k_end);
            }
            dc_compute<KIND, NT, GRAN>(st, nxt, qb, key0 + STEP, key_lo, k_end, pos, f, slope, biased);
        }
    } else {                                                         // a group of a wide head fills the registers
        for (; key0 < k_end; key0 += STEP) {
            dc_compute<KIND, NT, GRAN>(st, cur, qb, key0, key_lo, k_end, pos, f, slope, biased);
            if (key0 + STEP < k_end) {
                dc_load(cur, base, pages, key0 + STEP, a.c.num_pages);
                dc_pages(pages, a.c, trow, key0 + 2 * STEP, k_end);
            }
        }
    }
    // the four warps' results, merged in order
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float l = st.l[n][j];
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const int h = 8 * n + 2 * t + j;
            if (h >= heads) continue;
            float* mine = red_s + (size_t)(warp * heads + h) * REC;
            if (g == 0) mine[0] = st.seen >> (2 * n + j) & 1 ? st.m[n][j] : -INFINITY, mine[1] = l;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
                *reinterpret_cast<float2*>(mine + 4 + dc_dim(i, g, 0)) = make_float2(st.o[n][i][j], st.o[n][i][2 + j]);
        }
    __syncthreads();
    for (int idx = threadIdx.x; idx < heads * HD; idx += DC_THREADS) {
        const int h = idx / HD, d = idx % HD;
        float m = -INFINITY, l = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < DC_WARPS; ++w) m = fmaxf(m, red_s[(size_t)(w * heads + h) * REC]);
#pragma unroll
        for (int w = 0; w < DC_WARPS; ++w) {
            const float* rec = red_s + (size_t)(w * heads + h) * REC;
            l = q8_add_scaled(rec[1], q8_below(rec[0], m), l);
            acc = fmaf(rec[4 + d], q8_ex2(q8_below(rec[0], m)), acc);
        }
        const size_t at = (size_t)row * a.nH + head0 + h;
        float* rec = a.scratch + (((size_t)e * a.nH + head0 + h) * a.n_splits + run) * REC;
        if (runs == 1) {
            a.out[at * HD + d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
        } else {
            rec[4 + d] = acc;
            if (d == 0) rec[0] = m, rec[1] = l;
        }
        if (d == 0 && run == 0 && a.n_splits > 1) rec[2] = (float)runs;          // the merge asks the first record
    }
}

template <int KIND, int NT, int GRAN>
__global__ void __launch_bounds__(DC_THREADS, HD <= 64 && NT == 1 ? 3 : 2)
attn_decode_q8_kernel(const DcArgs a) {
    extern __shared__ float red_s[];                                 // [warp][head][REC]
    ng_pdl_trigger();
    const int segments = a.c.nKV * a.chunks;
    if (a.n_splits == 1) {
        const int e = blockIdx.x / segments, n = dc_turns(a, e);
        ng_pdl_wait();
        if (n) dc_piece<KIND, NT, GRAN>(a, red_s, e, blockIdx.x - e * segments, 0, n, 0, 1);
        return;
    }
    const int team = blockIdx.x / segments, segment = blockIdx.x - team * segments;
    DcShare sh = dc_share(a, team, gridDim.x / segments);
    ng_pdl_wait();
    for (int at = sh.first; at < sh.last && sh.e < a.n_entries;) {
        const int turns = dc_turns(a, sh.e), end = sh.before + dc_length(sh, turns);        // (entries without a single token have none)
        if (at < end) {
            const int turn0 = at - sh.before, turn1 = min(turns, sh.last - sh.before);
            const int t0 = sh.before / sh.each, t1 = (sh.before + turns - 1) / sh.each;
            if (at != sh.first) __syncthreads();                     // the piece before has been merged
            dc_piece<KIND, NT, GRAN>(a, red_s, sh.e, segment, turn0, turn1, team - t0, t1 - t0 + 1);
        }
        at = max(at, end);
        sh.before = end;
        ++sh.e;
    }
}

// ===================================================================================== portions
// Flash attention of prompt portions.  A row of a block is a (token, query head of the KV head): heads fastest, so that a short
// portion fills the block's PF_ROWS rows with the heads that share its keys, and a key tile is read and turned into float16 once for
// all of them.  64-key tiles: the codes of the next tile are requested into registers while this one is computed, then written to shared
// memory as float16 (two stages, one barrier a tile); scores, weights and sums as for single tokens, 16 rows a warp.
// For the heads that attention_q8_sm100.cu does not take, and what it refuses.  Bound by `mma.sync` and its ldmatrix loads (2,048 tokens, 32 / 8
// heads of 64: 97 us, there 42; 512 behind 32,768 496 and 180).
#define PF_WARPS 8
#define PF_THREADS (PF_WARPS * 32)
#define PF_ROWS (PF_WARPS * 16)
#define PF_KEYS 64
#define PF_LD (HD + 8)               // halves a row of the tile takes: 16-byte aligned, no bank met twice by ldmatrix
constexpr int PF_PIECES = PF_KEYS * HD / 16;                         // 16-byte pieces of a tile's K (and of its V)
constexpr int PF_EACH = (PF_PIECES + PF_THREADS - 1) / PF_THREADS;   // of a thread

struct PfSmem {
    uint16_t q[PF_ROWS][PF_LD];
    uint16_t k[2][PF_KEYS][PF_LD], v[2][PF_KEYS][PF_LD];
    float ks[2][PF_KEYS / 8], vl[2][PF_KEYS / 8], vi[2][PF_KEYS / 8];       // of each 8 keys: K's scale, V's log2 and reciprocal
    float f[PF_ROWS], slope[PF_ROWS];
};
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)));
}

struct PfArgs {
    Cache c;
    const bf16* q;
    const int *cu_q, *ctx_before;
    bf16* out;
    float* scratch;
    const float* slopes;
    int n_rows, n_entries, nH, window, skip_single;
    int n_splits;
    float scale;
};
struct PfTile {
    uint32_t k[PF_EACH][4], v[PF_EACH][4];
    float ks, vs;                                                    // threads 0 .. 7: of their 8 keys; vs -1: they have no page
};
__device__ __forceinline__ void pf_load(PfTile& r, const Cache& c, const int* trow, int key0, int key_lo, int k_end, int kvh) {
    const int mask = (1 << c.ps_log2) - 1;
#pragma unroll
    for (int n = 0; n < PF_EACH; ++n) {
        const int i = threadIdx.x + n * PF_THREADS, key = key0 + i / (HD / 16);
        int page = -1;
        if ((PF_PIECES % PF_THREADS == 0 || i < PF_PIECES) && key >= key_lo && key < k_end && (key >> c.ps_log2) < c.table_stride)
            page = trow[key >> c.ps_log2];
#pragma unroll
        for (int j = 0; j < 4; ++j) r.k[n][j] = r.v[n][j] = 0u;      // keys that no row sees: zeros (their codes may be NaN)
        if (page >= 0 && page < c.num_pages) {
            const size_t at = ((((size_t)page * c.nKV + kvh) << c.ps_log2) + (key & mask)) * HD + (i % (HD / 16)) * 16;
            ld_codes<16>(r.k[n], c.k + at);
            ld_codes<16>(r.v[n], c.v + at);
        }
    }
    r.ks = 1.f;
    r.vs = -1.f;
    if (threadIdx.x < PF_KEYS / 8) {
        const int key = key0 + 8 * threadIdx.x;
        int page = -1;
        if (key + 7 >= key_lo && key < k_end && (key >> c.ps_log2) < c.table_stride) page = trow[key >> c.ps_log2];
        if (page >= 0 && page < c.num_pages) {
            const size_t sc = (((size_t)page * c.nKV + kvh) << (c.ps_log2 - c.bl_log2)) + ((key & mask) >> c.bl_log2);
            r.ks = c.ks[sc];
            r.vs = c.vs[sc];
        }
    }
}
template <int KIND>
__device__ __forceinline__ void pf_store(PfSmem* sm, int s, const PfTile& r) {
#pragma unroll
    for (int n = 0; n < PF_EACH; ++n) {
        const int i = threadIdx.x + n * PF_THREADS;
        if (PF_PIECES % PF_THREADS != 0 && i >= PF_PIECES) break;
        const int key = i / (HD / 16), d = (i % (HD / 16)) * 16;
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) q8_to_half<KIND>(r.k[n][j], h[2 * j], h[2 * j + 1]);
        *reinterpret_cast<uint4*>(&sm->k[s][key][d]) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(&sm->k[s][key][d + 8]) = make_uint4(h[4], h[5], h[6], h[7]);
#pragma unroll
        for (int j = 0; j < 4; ++j) q8_to_half<KIND>(r.v[n][j], h[2 * j], h[2 * j + 1]);
        *reinterpret_cast<uint4*>(&sm->v[s][key][d]) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(&sm->v[s][key][d + 8]) = make_uint4(h[4], h[5], h[6], h[7]);
    }
    if (threadIdx.x < PF_KEYS / 8) {
        sm->ks[s][threadIdx.x] = r.ks;
        sm->vl[s][threadIdx.x] = r.vs < 0.f ? -INFINITY : q8_log2(r.vs);         // hidden
        sm->vi[s][threadIdx.x] = q8_recip(r.vs);                     // (1, times weights of 0)
    }
}

template <int KIND>
__global__ void __launch_bounds__(PF_THREADS, HD <= 64 ? 2 : 1)
attn_prefill_q8_kernel(const PfArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    PfSmem* sm = reinterpret_cast<PfSmem*>(smem_raw);
    ng_pdl_trigger();
    const int split = blockIdx.z, kvh = blockIdx.x, G = a.nH / a.c.nKV;
    const RowTile mine = row_tile(a.cu_q, a.n_entries, a.n_rows, G, PF_ROWS, a.skip_single, blockIdx.y);
    const int e = max(mine.e, 0), r0 = mine.first;
    const int q0 = a.cu_q[e], qlen = min(a.cu_q[e + 1], a.n_rows) - q0, ctx = a.ctx_before[e];
    ng_pdl_wait();
    if (mine.e < 0 || ctx < 0 || ctx > a.c.last_key) return;
    const int rows_here = min(PF_ROWS, qlen * G - r0);
    const int pos_first = ctx + r0 / G, pos_last = ctx + (r0 + rows_here - 1) / G;
    const int key_lo = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
    int tile0 = key_lo / PF_KEYS, tile1 = pos_last / PF_KEYS;        // inclusive
    if (a.n_splits > 1) {
        const int per = (tile1 - tile0 + a.n_splits) / a.n_splits;
        tile0 += split * per;
        tile1 = min(tile1, tile0 + per - 1);
    }
    const int k_end = pos_last + 1;
    const int* trow = a.c.table + (size_t)e * a.c.table_stride;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row_lo = warp * 16 + g, row_hi = row_lo + 8;

    PfTile next;
    if (tile0 <= tile1) pf_load(next, a.c, trow, tile0 * PF_KEYS, key_lo, k_end, kvh);
    // q -> shared memory as float16, a warp its 16 rows one after the other, each divided by a power of two
    const bf16* q = ng_after_wait(a.q);
    for (int i = 0; i < 16; ++i) {
        const int r = warp * 16 + i;
        const bool live = r < rows_here;
        const int token = (r0 + min(r, rows_here - 1)) / G, head = kvh * G + (r0 + min(r, rows_here - 1)) - token * G;
        const bf16* src = q + ((size_t)(q0 + token) * a.nH + head) * HD;
        uint32_t w[(HD + 63) / 64];
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < (HD + 63) / 64; ++j) {
            const int d = 2 * lane + 64 * j;
            w[j] = live && d < HD ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
            const float x = fabsf(__uint_as_float(w[j] << 16)), y = fabsf(__uint_as_float(w[j] & 0xffff0000u));
            if (x < INFINITY) top = fmaxf(top, x);
            if (y < INFINITY) top = fmaxf(top, y);
        }
        const int ex = q_exponent(ng_warp_max(top));
        const float f = pow2_any(-ex);
#pragma unroll
        for (int j = 0; j < (HD + 63) / 64; ++j) {
            const int d = 2 * lane + 64 * j;
            if (d < HD) *reinterpret_cast<uint32_t*>(&sm->q[r][d]) = pack_f16(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xffff0000u) * f);
        }
        if (lane == 0) {
            sm->f[r] = a.scale * LOG2E * pow2_any(ex);
            sm->slope[r] = a.slopes ? a.slopes[head] * LOG2E : 0.f;
        }
    }
    __syncwarp();
    const float f_lo = sm->f[row_lo], f_hi = sm->f[row_hi], slope_lo = sm->slope[row_lo], slope_hi = sm->slope[row_hi];
    const int pos_lo = ctx + (r0 + min(row_lo, rows_here - 1)) / G, pos_hi = ctx + (r0 + min(row_hi, rows_here - 1)) / G;
    // this warp's first and last position: tiles between need no mask
    const int w_first = ctx + (r0 + min(warp * 16, rows_here - 1)) / G, w_last = ctx + (r0 + min(warp * 16 + 15, rows_here - 1)) / G;

    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
    bool high = false;                                               // (Q8_HIGH)
    constexpr bool Q_HELD = HD <= 64;
    uint32_t qa[Q_HELD ? HD / 16 : 1][4];
    if constexpr (Q_HELD)
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) ldmatrix_x4(qa[i], &sm->q[warp * 16 + (lane & 15)][i * 16 + 8 * (lane >> 4)]);

    for (int tile = tile0; tile <= tile1; ++tile) {
        const int s = (tile - tile0) & 1, key0 = tile * PF_KEYS;
        pf_store<KIND>(sm, s, next);
        __syncthreads();                                             // (stage s was last read two tiles ago: every warp has passed a barrier since)
        if (tile < tile1) pf_load(next, a.c, trow, key0 + PF_KEYS, key_lo, k_end, kvh);
        if (key0 > w_last || (a.window > 0 && key0 + PF_KEYS - 1 <= w_first - a.window)) continue;      // no row of the warp sees a key of it
        float sc[PF_KEYS / 8][4];
#pragma unroll
        for (int i = 0; i < PF_KEYS / 8; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll
        for (int kb = 0; kb < HD / 16; ++kb) {
            uint32_t qq[4];
            if constexpr (!Q_HELD) ldmatrix_x4(qq, &sm->q[warp * 16 + (lane & 15)][kb * 16 + 8 * (lane >> 4)]);
            else { qq[0] = qa[kb][0]; qq[1] = qa[kb][1]; qq[2] = qa[kb][2]; qq[3] = qa[kb][3]; }
#pragma unroll
            for (int np = 0; np < PF_KEYS / 16; ++np) {
                uint32_t b[4];
                ldmatrix_x4(b, &sm->k[s][np * 16 + (lane & 7) + 8 * (lane >> 4)][kb * 16 + 8 * ((lane >> 3) & 1)]);
                mma_f16(sc[2 * np], qq, b[0], b[1]);
                mma_f16(sc[2 * np + 1], qq, b[2], b[3]);
            }
        }
        const bool whole = key0 + PF_KEYS - 1 <= w_first && (a.window <= 0 || key0 > w_last - a.window);
        float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < PF_KEYS / 8; ++nt) {
            const float ks = sm->ks[s][nt], lg = sm->vl[s][nt], fa = f_lo * ks, fb = f_hi * ks;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                sc[nt][j] = fmaf(sc[nt][j], fa, lg);
                sc[nt][2 + j] = fmaf(sc[nt][2 + j], fb, lg);
                if (!whole || a.slopes) {
                    const int key = key0 + nt * 8 + 2 * t + j;
                    const bool ok_lo = key <= pos_lo && (a.window <= 0 || key > pos_lo - a.window);
                    const bool ok_hi = key <= pos_hi && (a.window <= 0 || key > pos_hi - a.window);
                    sc[nt][j] = ok_lo ? fmaf(-slope_lo, (float)(pos_lo - key), sc[nt][j]) : -INFINITY;
                    sc[nt][2 + j] = ok_hi ? fmaf(-slope_hi, (float)(pos_hi - key), sc[nt][2 + j]) : -INFINITY;
                }
                mx_lo = fmaxf(mx_lo, sc[nt][j]);
                mx_hi = fmaxf(mx_hi, sc[nt][2 + j]);
            }
        }
        if (__any_sync(0xffffffffu, mx_lo > m_lo + 8.f || mx_hi > m_hi + 8.f || m_lo == -INFINITY || m_hi == -INFINITY)) {
#pragma unroll
            for (int x = 1; x <= 2; x <<= 1) {
                mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, x));
                mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, x));
            }
            const float n_lo = fmaxf(m_lo, mx_lo), n_hi = fmaxf(m_hi, mx_hi);
            const float c_lo = n_lo == -INFINITY ? 1.f : q8_ex2(m_lo - n_lo), c_hi = n_hi == -INFINITY ? 1.f : q8_ex2(m_hi - n_hi);
            high = high || __any_sync(0xffffffffu, sm->vl[s][lane & 7] > Q8_HIGH);
            l_lo = q8_add_scaled(l_lo, q8_below(m_lo, n_lo), 0.f);
            l_hi = q8_add_scaled(l_hi, q8_below(m_hi, n_hi), 0.f);
            m_lo = n_lo;
            m_hi = n_hi;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) { o[i][0] *= c_lo; o[i][1] *= c_lo; o[i][2] *= c_hi; o[i][3] *= c_hi; }
        }
        const float ref_lo = m_lo == -INFINITY ? 0.f : m_lo, ref_hi = m_hi == -INFINITY ? 0.f : m_hi;
        uint32_t p[PF_KEYS / 16][4];
        const float lg8 = sm->vl[s][lane & 7];                       // (minus infinity for keys that are hidden)
        if (__any_sync(0xffffffffu, (lg8 < Q8_LOW && lg8 != -INFINITY) || high))
#pragma unroll
            for (int nt = 0; nt < PF_KEYS / 8; ++nt) {               // in place of what is added below
                const float lg = sm->vl[s][nt] == -INFINITY ? 0.f : sm->vl[s][nt], inv = sm->vi[s][nt];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l_lo += q8_ex2(sc[nt][j] - ref_lo - lg) - q8_ex2(sc[nt][j] - ref_lo) * inv;
                    l_hi += q8_ex2(sc[nt][2 + j] - ref_hi - lg) - q8_ex2(sc[nt][2 + j] - ref_hi) * inv;
                }
            }
#pragma unroll
        for (int nt = 0; nt < PF_KEYS / 8; ++nt) {
            const float p0 = q8_ex2(sc[nt][0] - ref_lo), p1 = q8_ex2(sc[nt][1] - ref_lo);
            const float p2 = q8_ex2(sc[nt][2] - ref_hi), p3 = q8_ex2(sc[nt][3] - ref_hi);
            const float inv = sm->vi[s][nt];
            l_lo = fmaf(p0 + p1, inv, l_lo);
            l_hi = fmaf(p2 + p3, inv, l_hi);
            p[nt >> 1][(nt & 1) * 2 + 0] = pack_f16(p0, p1);
            p[nt >> 1][(nt & 1) * 2 + 1] = pack_f16(p2, p3);
        }
#pragma unroll
        for (int kk = 0; kk < PF_KEYS / 16; ++kk)
#pragma unroll
            for (int dp = 0; dp < HD / 16; ++dp) {
                uint32_t b[4];
                ldmatrix_x4_trans(b, &sm->v[s][kk * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)][dp * 16 + 8 * (lane >> 4)]);
                mma_f16(o[2 * dp], p[kk], b[0], b[1]);
                mma_f16(o[2 * dp + 1], p[kk], b[2], b[3]);
            }
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        l_lo += __shfl_xor_sync(0xffffffffu, l_lo, x);
        l_hi += __shfl_xor_sync(0xffffffffu, l_hi, x);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = half ? row_hi : row_lo;
        if (r >= rows_here) continue;
        const int token = (r0 + r) / G, head = kvh * G + (r0 + r) - token * G;
        const size_t at = (size_t)(q0 + token) * a.nH + head;
        const float l = half ? l_hi : l_lo;
        if (a.n_splits > 1) {
            float* rec = a.scratch + (at * a.n_splits + split) * REC;
            if (t == 0) rec[0] = half ? m_hi : m_lo, rec[1] = l;
            if (l == 0.f) continue;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
                *reinterpret_cast<float2*>(rec + 4 + i * 8 + 2 * t) = make_float2(o[i][2 * half], o[i][2 * half + 1]);
        } else {
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
                *reinterpret_cast<__nv_bfloat162*>(a.out + at * HD + i * 8 + 2 * t) = __floats2bfloat162_rn(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
        }
    }
}

// ===================================================================================== host
// blocks of the kernel that the current device holds at once (with the most shared memory it may ask for)
template <typename K>
static int dc_slots(std::atomic<int>* known, K kernel) {
    int device = 0, sms = 0, each = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 0;
    int n = known[device & 63].load(std::memory_order_relaxed);
    if (n) return n;
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, DC_THREADS, attr.maxDynamicSharedSizeBytes) != cudaSuccess)
        return 0;
    n = sms * (each > 0 ? each : 1);
    known[device & 63].store(n, std::memory_order_relaxed);
    return n;
}

// scratch (n_splits > 1): n_entries * n_heads * n_splits * REC floats, 16-byte aligned
NG_EXPORT int ng_attn_decode_q8(const NgAttnQ8* call, cudaStream_t stream) {
    const NgAttnQ8& c = *call;
    const int n_entries = c.n_entries, nKV = c.n_kv, nH = c.n_heads, n_splits = c.n_splits, kind = c.kind, block = c.block;
    if (n_entries <= 0 || c.n_rows <= 0) return NG_OK;
    DcArgs a;
    if (!attn_q8_args(c, a.c) || n_splits > 65535 || n_entries > 65535 || ((uintptr_t)c.q & 7) || ((uintptr_t)c.out & 3)) return NG_BAD_SIZE;
    const int G = nH / nKV;
    a.q = (const bf16*)c.q; a.cu_q = c.cu_q; a.ctx_before = c.ctx_before; a.out = (bf16*)c.out; a.scratch = c.scratch; a.slopes = c.slopes;
    a.n_rows = c.n_rows; a.n_entries = n_entries; a.nH = nH; a.window = c.window; a.n_splits = n_splits; a.scale = c.scale;
    const int nt = G > 8 ? DC_NT_MAX : 1;
    a.chunks = (G + 8 * nt - 1) / (8 * nt);
    const int segments = nKV * a.chunks;
    // blocks, and all turns rounded up to whole shares, are counted in 31 bits
    if ((long long)nKV * a.chunks * n_entries > 0x7fffffff || n_entries * (((long long)c.table_stride * c.page_size / TURN + 2) * 2) > 0x7fffffff)
        return NG_BAD_SIZE;
#define DC_GO(KIND, NT, GRAN)                                                                                                         \
    do {                                                                                                                              \
        static std::atomic<unsigned long long> once{0};                                                                               \
        static std::atomic<int> slots[64];                                                                                            \
        constexpr auto kernel = attn_decode_q8_kernel<KIND, NT, GRAN>;                                                                \
        if (!ng_allow_smem(once, kernel, DC_WARPS * 8 * NT * REC * (int)sizeof(float))) return NG_LAUNCH_FAILED;                      \
        const int smem = DC_WARPS * (G < 8 * NT ? G : 8 * NT) * REC * (int)sizeof(float);                                             \
        const int room = n_splits > 1 ? dc_slots(slots, kernel) : 1;                                                                  \
        if (room <= 0) return NG_LAUNCH_FAILED;                                                                                       \
        const int teams = room / segments > 1 ? room / segments : 1;                                                                  \
        NG_LAUNCH((kernel), dim3(n_splits > 1 ? teams * segments : n_entries * segments), DC_THREADS, smem, stream, a);                                  \
    } while (0)
#define DC_KINDS(NT, GRAN) do { if (kind == NG_Q8_E4M3) DC_GO(NG_Q8_E4M3, NT, GRAN); else DC_GO(NG_Q8_INT8, NT, GRAN); } while (0)
    if (nt == 1 && block >= 16) DC_KINDS(1, 16);
    else if (nt == 1) DC_KINDS(1, 8);
    else if (block >= 16) DC_KINDS(DC_NT_MAX, 16);
    else DC_KINDS(DC_NT_MAX, 8);
    if (n_splits > 1) return q8_merge(c, a.c, true, 1, stream);
    return ng_launch_status();
}

// scratch (n_splits > 1): n_rows * n_heads * n_splits * REC floats, 16-byte aligned
NG_EXPORT int ng_attn_prefill_q8(const NgAttnQ8* call, cudaStream_t stream) {
    const NgAttnQ8& c = *call;
    const int kind = c.kind;
    if (c.n_entries <= 0 || c.n_rows <= 0 || c.max_q <= 0) return NG_OK;
    PfArgs a;
    if (!attn_q8_args(c, a.c) || c.n_splits > 65535 || (((uintptr_t)c.q | (uintptr_t)c.out) & 3)) return NG_BAD_SIZE;
    const long long tiles = q8_row_tiles(c, PF_ROWS);
    if (tiles > 65535) return NG_BAD_SIZE;
    if (tiles <= 0) return NG_OK;                              // (one row, and single tokens are left out)
    a.q = (const bf16*)c.q; a.cu_q = c.cu_q; a.ctx_before = c.ctx_before; a.out = (bf16*)c.out; a.scratch = c.scratch; a.slopes = c.slopes;
    a.n_rows = c.n_rows; a.n_entries = c.n_entries; a.nH = c.n_heads; a.window = c.window; a.n_splits = c.n_splits; a.skip_single = c.skip_single;
    a.scale = c.scale;
    const dim3 grid(c.n_kv, (unsigned)tiles, c.n_splits);
#define PF_GO(KIND)                                                                                                  \
    do {                                                                                                             \
        static std::atomic<unsigned long long> once{0};                                                              \
        if (!ng_allow_smem(once, attn_prefill_q8_kernel<KIND>, (int)sizeof(PfSmem))) return NG_LAUNCH_FAILED;        \
        NG_LAUNCH((attn_prefill_q8_kernel<KIND>), grid, PF_THREADS, sizeof(PfSmem), stream, a);                      \
    } while (0)
    if (kind == NG_Q8_E4M3) PF_GO(NG_Q8_E4M3);
    else PF_GO(NG_Q8_INT8);
    if (c.n_splits > 1) return q8_merge(c, a.c, false, c.skip_single ? 2 : 1, stream);
    return ng_launch_status();
}
