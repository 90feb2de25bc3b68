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
// whose values are small has small weights, not small values, and the sum over the codes never leaves float16's range.
#include "ng_q8.cuh"

#ifndef NG_HEAD_DIM
#error "compile with -DNG_HEAD_DIM=<head size>"
#endif
#define HD NG_HEAD_DIM
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 in [16, 256]");
#define LOG2E 1.4426950408889634f
#define REC (HD + 4)            // floats of a run's record: reference point, sum, two unused (the row starts on 16 bytes), row in codes

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float ex2(float x) {          // 2 ulp; -inf -> 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// BYTES of codes from a page; no line of the first-level cache is taken (they are read once).  Not moved above the wait.
template <int BYTES>
__device__ __forceinline__ void ld_codes(uint32_t* w, const unsigned char* p) {
    if constexpr (BYTES == 16)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p) : "memory");
    else if constexpr (BYTES == 8)
        asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p) : "memory");
    else if constexpr (BYTES == 4)
        asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p) : "memory");
    else
        asm volatile("{\n\t.reg .u16 h;\n\tld.global.L1::no_allocate.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(w[0]) : "l"(p) : "memory");
}

// The power of two that a row of q is divided by (its largest value becomes 1 to 2): exponent of the row's largest finite value.
__device__ __forceinline__ int q_exponent(float top) { return min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127); }
__device__ __forceinline__ float pow2_any(int e) { return q8_pow2(min(max(e, -126), 127)); }

struct Cache {
    const unsigned char *k, *v;          // [pages, nKV, page, HD]
    const float *ks, *vs;                // [pages, nKV, page / block]
    const int* table;
    int table_stride, num_pages, nKV, ps_log2, bl_log2;
};

// ===================================================================================== single tokens
// A block owns one (entry, 16 or fewer query heads of one KV head, run of the keys).  Its four warps take groups of 16 * SUB keys in
// turn, each on its own (no barrier until the end): the heads are the rows of one MMA tile, the contraction index of q.c and the output
// dimension are permuted so that a lane reads contiguous bytes, and K and V come from memory into the registers they are used
// from, the next group's requested before this group is computed.  Nothing passes through shared memory but the four warps' results.
//
// Bound by the codes' bytes.  A lane's words of V hold four keys' codes of one dimension apart; two byte permutations a pair of
// words put a pair of keys beside each other, as the MMA wants them.
#define DC_WARPS 4
#define DC_THREADS (DC_WARPS * 32)
constexpr int W = HD % 64 == 0 ? 16 : HD % 32 == 0 ? 8 : 4;        // bytes of a key that a lane takes at once (of a value row: half of it)
constexpr int NC = HD / (4 * W);                                    // such pieces a row has for it
constexpr int SUB = HD <= 64 ? 2 : 1;                               // 16-key tiles a group has
constexpr int GROUP = 16 * SUB;

struct DcGroup {
    uint32_t k[SUB][2][NC * W / 4];          // keys g and 8 + g of the tile
    uint32_t v[SUB][4][NC * ((W / 2 + 3) / 4)];       // keys 2t, 2t+1, 8+2t, 8+2t+1
    float ks[SUB][2], vs[SUB][2];            // of the tile's halves
};

// Keys key0 .. key0 + GROUP - 1 of the block's run.  Halves (8 keys: one page, one block) that have no key of the run, and pages
// that are not there, give zeros.
__device__ __forceinline__ void dc_load(DcGroup& r, const Cache& c, const int* trow, int key0, int k_end, int kvh) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    int page[SUB][2];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int key = key0 + 16 * s + 8 * h;
            page[s][h] = key < k_end && (key >> c.ps_log2) < c.table_stride ? trow[key >> c.ps_log2] : -1;
        }
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int slot = (key0 + 16 * s + 8 * h) & ((1 << c.ps_log2) - 1);
            const bool ok = page[s][h] >= 0 && page[s][h] < c.num_pages;
            const size_t slab = (size_t)(ok ? page[s][h] : 0) * c.nKV + kvh;
            const size_t at = ((slab << c.ps_log2) + slot) * HD;
            const size_t sc = (slab << (c.ps_log2 - c.bl_log2)) + (slot >> c.bl_log2);
            r.ks[s][h] = ok ? c.ks[sc] : 1.f;
            r.vs[s][h] = ok ? c.vs[sc] : 1.f;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
#pragma unroll
                for (int i = 0; i < W / 4; ++i) r.k[s][h][n * (W / 4) + i] = 0;
                if (ok) ld_codes<W>(&r.k[s][h][n * (W / 4)], c.k + at + (size_t)g * HD + n * 4 * W + t * W);
            }
            constexpr int VW = (W / 2 + 3) / 4;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int n = 0; n < NC; ++n) {
#pragma unroll
                    for (int i = 0; i < VW; ++i) r.v[s][2 * h + j][n * VW + i] = 0;
                    if (ok) ld_codes<W / 2>(&r.v[s][2 * h + j][n * VW], c.v + at + (size_t)(2 * t + j) * HD + n * 4 * W + g * (W / 2));
                }
        }
}

struct DcState {
    float o[HD / 8][4], m_lo, m_hi, l_lo, l_hi;
};

// One group into the warp's state.  f_lo, f_hi: what the raw products of the lane's two rows are multiplied by (base 2).
template <int KIND>
__device__ __forceinline__ void dc_compute(DcState& st, const DcGroup& r, const uint32_t (&qa)[HD / 16][4], int key0, int key_lo, int k_end,
                                           int pos, float f_lo, float f_hi, float slope_lo, float slope_hi) {
    const int t = threadIdx.x & 3;
    float sc[SUB][2][4];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sc[s][h][0] = sc[s][h][1] = sc[s][h][2] = sc[s][h][3] = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                uint32_t b0, b1;
                q8_to_half<KIND>(r.k[s][h][i], b0, b1);
                mma_f16(sc[s][h], qa[i], b0, b1);
            }
        }
    const bool whole = key0 >= key_lo && key0 + GROUP <= k_end;
    float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float a = f_lo * r.ks[s][h], b = f_hi * r.ks[s][h], lg = q8_log2(r.vs[s][h]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int key = key0 + 16 * s + 8 * h + 2 * t + j;
                const bool ok = whole || (key >= key_lo && key < k_end);
                const float away = (float)(pos - key);
                sc[s][h][j] = ok ? fmaf(-slope_lo, away, fmaf(sc[s][h][j], a, lg)) : -INFINITY;
                sc[s][h][2 + j] = ok ? fmaf(-slope_hi, away, fmaf(sc[s][h][2 + j], b, lg)) : -INFINITY;
                mx_lo = fmaxf(mx_lo, sc[s][h][j]);
                mx_hi = fmaxf(mx_hi, sc[s][h][2 + j]);
            }
        }
    // the reference point follows the maximum lazily: weights may reach 2^8 before the sums are rescaled
    if (__any_sync(0xffffffffu, mx_lo > st.m_lo + 8.f || mx_hi > st.m_hi + 8.f || st.m_lo == -INFINITY || st.m_hi == -INFINITY)) {
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, x));
            mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, x));
        }
        const float n_lo = fmaxf(st.m_lo, mx_lo), n_hi = fmaxf(st.m_hi, mx_hi);
        const float c_lo = n_lo == -INFINITY ? 1.f : ex2(st.m_lo - n_lo), c_hi = n_hi == -INFINITY ? 1.f : ex2(st.m_hi - n_hi);
        st.m_lo = n_lo;
        st.m_hi = n_hi;
        st.l_lo *= c_lo;
        st.l_hi *= c_hi;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) { st.o[i][0] *= c_lo; st.o[i][1] *= c_lo; st.o[i][2] *= c_hi; st.o[i][3] *= c_hi; }
    }
    const float ref_lo = st.m_lo == -INFINITY ? 0.f : st.m_lo, ref_hi = st.m_hi == -INFINITY ? 0.f : st.m_hi;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
        uint32_t pa[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float p0 = ex2(sc[s][h][0] - ref_lo), p1 = ex2(sc[s][h][1] - ref_lo);
            const float p2 = ex2(sc[s][h][2] - ref_hi), p3 = ex2(sc[s][h][3] - ref_hi);
            const float inv = q8_recip(r.vs[s][h]);
            st.l_lo = fmaf(p0 + p1, inv, st.l_lo);
            st.l_hi = fmaf(p2 + p3, inv, st.l_hi);
            pa[2 * h] = pack_f16(p0, p1);
            pa[2 * h + 1] = pack_f16(p2, p3);
        }
        uint32_t v[4][sizeof(r.v[0][0]) / 4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // a key that no row sees has a weight of 0, but its codes may be NaN
            const int key = key0 + 16 * s + 8 * (j >> 1) + 2 * t + (j & 1);
            const bool ok = whole || (key >= key_lo && key < k_end);
#pragma unroll
            for (int i = 0; i < (int)(sizeof(r.v[0][0]) / 4); ++i) v[j][i] = ok ? r.v[s][j][i] : 0u;
        }
        if constexpr (W >= 8) {
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {                     // a word: four dimensions
                uint32_t b0[4], b1[4];
                q8_to_half<KIND>(__byte_perm(v[0][i], v[1][i], 0x5140), b0[0], b0[1]);
                q8_to_half<KIND>(__byte_perm(v[0][i], v[1][i], 0x7362), b0[2], b0[3]);
                q8_to_half<KIND>(__byte_perm(v[2][i], v[3][i], 0x5140), b1[0], b1[1]);
                q8_to_half<KIND>(__byte_perm(v[2][i], v[3][i], 0x7362), b1[2], b1[3]);
#pragma unroll
                for (int d = 0; d < 4; ++d) mma_f16(st.o[4 * i + d], pa, b0[d], b1[d]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i) {                          // two dimensions in a word's lower half
                uint32_t b0[2], b1[2];
                q8_to_half<KIND>(__byte_perm(v[0][i], v[1][i], 0x5140), b0[0], b0[1]);
                q8_to_half<KIND>(__byte_perm(v[2][i], v[3][i], 0x5140), b1[0], b1[1]);
#pragma unroll
                for (int d = 0; d < 2; ++d) mma_f16(st.o[2 * i + d], pa, b0[d], b1[d]);
            }
        }
    }
}
// the head's dimension of column n (0..7) of MMA tile i
__device__ __forceinline__ int dc_dim(int i, int n) {
    constexpr int PER = W / 2;                                       // dimensions a lane group has of a piece
    return (i / PER) * 8 * PER + n * PER + i % PER;
}

struct DcArgs {
    Cache c;
    const bf16* q;
    const int *cu_q, *ctx_before;
    bf16* out;
    float* scratch;
    const float* slopes;
    int n_rows, nH, chunks, window, n_splits, keys_per_split;
    float scale;
};

template <int KIND>
__global__ void __launch_bounds__(DC_THREADS, HD <= 64 ? 4 : HD <= 128 ? 3 : 2)
attn_decode_q8_kernel(const DcArgs a) {
    extern __shared__ float red_s[];                                 // [warp][head][REC]
    ng_pdl_trigger();
    const int e = blockIdx.y, kvh = blockIdx.x / a.chunks, split = blockIdx.z;
    const int row = a.cu_q[e], n_here = a.cu_q[e + 1] - row, pos = a.ctx_before[e];
    ng_pdl_wait();
    if (n_here != 1 || row < 0 || row >= a.n_rows || pos < 0) return;
    const int G = a.nH / a.c.nKV, h0 = (blockIdx.x - kvh * a.chunks) * 16, heads = min(16, G - h0);
    const int head0 = kvh * G + h0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int key_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int k_begin = (key_lo & ~(GROUP - 1)) + split * a.keys_per_split;
    // the last run takes what is left: a caller's bound on the keys that is too low costs time, not keys
    const int k_end = split == a.n_splits - 1 ? pos + 1 : min(pos + 1, k_begin + a.keys_per_split);
    const int* trow = a.c.table + (size_t)e * a.c.table_stride;

    DcGroup cur, nxt;
    int key0 = k_begin + warp * GROUP;
    if (key0 < k_end) dc_load(cur, a.c, trow, key0, k_end, kvh);

    // rows of the MMA tile: the block's heads (rows beyond them are zero), each divided by a power of two
    uint32_t qa[HD / 16][4];
    float f_lo, f_hi, slope_lo = 0.f, slope_hi = 0.f;
    {
        const bf16* q = ng_after_wait(a.q) + ((size_t)row * a.nH + head0) * HD;
        uint2 lo[HD / 16], hi[HD / 16];
        float top_lo = 0.f, top_hi = 0.f;
        auto top_of = [](uint2 w, float top) {
            const uint32_t x[4] = {w.x << 16, w.x & 0xffff0000u, w.y << 16, w.y & 0xffff0000u};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = fabsf(__uint_as_float(x[i]));
                top = v < INFINITY ? fmaxf(top, v) : top;
            }
            return top;
        };
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            const int d = (i / (W / 4)) * 4 * W + t * W + (i % (W / 4)) * 4;
            lo[i] = g < heads ? *reinterpret_cast<const uint2*>(q + (size_t)g * HD + d) : make_uint2(0u, 0u);
            hi[i] = g + 8 < heads ? *reinterpret_cast<const uint2*>(q + (size_t)(g + 8) * HD + d) : make_uint2(0u, 0u);
            top_lo = top_of(lo[i], top_lo);
            top_hi = top_of(hi[i], top_hi);
        }
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            top_lo = fmaxf(top_lo, __shfl_xor_sync(0xffffffffu, top_lo, x));
            top_hi = fmaxf(top_hi, __shfl_xor_sync(0xffffffffu, top_hi, x));
        }
        const int e_lo = q_exponent(top_lo), e_hi = q_exponent(top_hi);
        const float d_lo = pow2_any(-e_lo), d_hi = pow2_any(-e_hi);
        f_lo = a.scale * LOG2E * pow2_any(e_lo);
        f_hi = a.scale * LOG2E * pow2_any(e_hi);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            qa[i][0] = pack_f16(__uint_as_float(lo[i].x << 16) * d_lo, __uint_as_float(lo[i].x & 0xffff0000u) * d_lo);
            qa[i][2] = pack_f16(__uint_as_float(lo[i].y << 16) * d_lo, __uint_as_float(lo[i].y & 0xffff0000u) * d_lo);
            qa[i][1] = pack_f16(__uint_as_float(hi[i].x << 16) * d_hi, __uint_as_float(hi[i].x & 0xffff0000u) * d_hi);
            qa[i][3] = pack_f16(__uint_as_float(hi[i].y << 16) * d_hi, __uint_as_float(hi[i].y & 0xffff0000u) * d_hi);
        }
        if (a.slopes && g < heads) slope_lo = a.slopes[head0 + g] * LOG2E;
        if (a.slopes && g + 8 < heads) slope_hi = a.slopes[head0 + g + 8] * LOG2E;
    }
    DcState st;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) st.o[i][0] = st.o[i][1] = st.o[i][2] = st.o[i][3] = 0.f;
    st.m_lo = st.m_hi = -INFINITY;
    st.l_lo = st.l_hi = 0.f;
    constexpr int STEP = DC_WARPS * GROUP;
    if constexpr (HD <= 128) {
        for (; key0 < k_end; key0 += 2 * STEP) {
            if (key0 + STEP < k_end) dc_load(nxt, a.c, trow, key0 + STEP, k_end, kvh);
            dc_compute<KIND>(st, cur, qa, key0, key_lo, k_end, pos, f_lo, f_hi, slope_lo, slope_hi);
            if (key0 + STEP >= k_end) break;
            if (key0 + 2 * STEP < k_end) dc_load(cur, a.c, trow, key0 + 2 * STEP, k_end, kvh);
            dc_compute<KIND>(st, nxt, qa, key0 + STEP, key_lo, k_end, pos, f_lo, f_hi, slope_lo, slope_hi);
        }
    } else {                                                         // a group of a wide head fills the registers
        for (; key0 < k_end; key0 += STEP) {
            dc_compute<KIND>(st, cur, qa, key0, key_lo, k_end, pos, f_lo, f_hi, slope_lo, slope_hi);
            if (key0 + STEP < k_end) dc_load(cur, a.c, trow, key0 + STEP, k_end, kvh);
        }
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        st.l_lo += __shfl_xor_sync(0xffffffffu, st.l_lo, x);
        st.l_hi += __shfl_xor_sync(0xffffffffu, st.l_hi, x);
    }
    // the four warps' results, merged in order
    float* mine = red_s + (size_t)(warp * heads + g) * REC;
    if (g < heads) {
        if (t == 0) mine[0] = st.m_lo, mine[1] = st.l_lo;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
            mine[4 + dc_dim(i, 2 * t)] = st.o[i][0];
            mine[4 + dc_dim(i, 2 * t + 1)] = st.o[i][1];
        }
    }
    if (g + 8 < heads) {
        mine += 8 * REC;
        if (t == 0) mine[0] = st.m_hi, mine[1] = st.l_hi;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
            mine[4 + dc_dim(i, 2 * t)] = st.o[i][2];
            mine[4 + dc_dim(i, 2 * t + 1)] = st.o[i][3];
        }
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
            const float f = rec[0] == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : ex2(rec[0] - m);       // (a warp that met only NaN kept its sums)
            l = fmaf(rec[1], f, l);
            acc = fmaf(rec[4 + d], f, acc);
        }
        const size_t at = (size_t)row * a.nH + head0 + h;
        if (a.n_splits == 1) {
            a.out[at * HD + d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
        } else {
            float* rec = a.scratch + (at * a.n_splits + split) * REC;
            rec[4 + d] = acc;
            if (d == 0) rec[0] = m, rec[1] = l;
        }
    }
}

// out[row, head] = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over the runs s, in ascending order within each of GROUPS
// groups of them, then the groups.  A block has a (row, head); its rows are the entries' single tokens, or (portions) all rows of the
// entries that bring more.
template <int GROUPS>
__global__ void __launch_bounds__(GROUPS * HD)
attn_q8_merge_kernel(const float* __restrict__ scratch, const int* __restrict__ cu_q, bf16* __restrict__ out, int nH, int n_splits,
                     int n_rows, int least, int most) {
    ng_pdl_trigger();
    const int e = blockIdx.y, head = blockIdx.x;
    const int q0 = cu_q[e], n = cu_q[e + 1] - q0;
    ng_pdl_wait();
    if (n < least || n > most) return;
    scratch = ng_after_wait(scratch);
    const int d = threadIdx.x % HD, g = threadIdx.x / HD;
    __shared__ float part[GROUPS][HD], part_l[GROUPS];
    for (int r = q0 + blockIdx.z; r < min(q0 + n, n_rows); r += gridDim.z) {
        const float* rec = scratch + ((size_t)r * nH + head) * n_splits * REC;
        float m = -INFINITY;
        for (int s = 0; s < n_splits; ++s) m = fmaxf(m, rec[(size_t)s * REC]);
        float l = 0.f, acc = 0.f;
#pragma unroll 4
        for (int s = g; s < n_splits; s += GROUPS) {
            const float ms = rec[(size_t)s * REC], ls = rec[(size_t)s * REC + 1];
            const float f = ms == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : ex2(ms - m);
            l = fmaf(ls, f, l);
            acc = fmaf(ls == 0.f ? 0.f : rec[(size_t)s * REC + 4 + d], f, acc);       // (an empty run wrote no row)
        }
        if constexpr (GROUPS > 1) {
            __syncthreads();
            part[g][d] = acc;
            if (d == 0) part_l[g] = l;
            __syncthreads();
            if (g == 0)
#pragma unroll
                for (int k = 1; k < GROUPS; ++k) {
                    l += part_l[k];
                    acc += part[k][d];
                }
        }
        if (g == 0) out[((size_t)r * nH + head) * HD + d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
    }
}

// ===================================================================================== portions
// Flash attention of prompt portions.  A row of a block is a (token, query head of the KV head): heads fastest, so that a short
// portion fills the block's PF_ROWS rows with the heads that share its keys, and a key tile is read and turned into float16 once for
// all of them.  64-key tiles: the codes of the next tile are requested into registers while this one is computed, then written to shared
// memory as float16 (two stages, one barrier a tile); scores, weights and sums as for single tokens, 16 rows a warp.
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
    int n_rows, nH, window, n_splits, skip_single;
    float scale;
};
struct PfTile {
    uint32_t k[PF_EACH][4], v[PF_EACH][4];
    float ks, vs;                                                    // threads 0 .. 7: of their 8 keys
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
    r.ks = r.vs = 1.f;
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
        sm->vl[s][threadIdx.x] = q8_log2(r.vs);
        sm->vi[s][threadIdx.x] = q8_recip(r.vs);
    }
}

template <int KIND>
__global__ void __launch_bounds__(PF_THREADS, HD <= 64 ? 2 : 1)
attn_prefill_q8_kernel(const PfArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    PfSmem* sm = reinterpret_cast<PfSmem*>(smem_raw);
    ng_pdl_trigger();
    // heads fastest, row tiles from the last down: the blocks with the most keys start first
    const int e = blockIdx.z / a.n_splits, split = blockIdx.z - e * a.n_splits, kvh = blockIdx.x;
    const int q0 = a.cu_q[e], qlen = min(a.cu_q[e + 1], a.n_rows) - q0, ctx = a.ctx_before[e];
    ng_pdl_wait();
    const int G = a.nH / a.c.nKV;
    const int r0 = (gridDim.y - 1 - blockIdx.y) * PF_ROWS;
    if (q0 < 0 || ctx < 0 || r0 >= qlen * G || (a.skip_single && a.cu_q[e + 1] - q0 == 1)) return;
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
            const float c_lo = n_lo == -INFINITY ? 1.f : ex2(m_lo - n_lo), c_hi = n_hi == -INFINITY ? 1.f : ex2(m_hi - n_hi);
            m_lo = n_lo;
            m_hi = n_hi;
            l_lo *= c_lo;
            l_hi *= c_hi;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) { o[i][0] *= c_lo; o[i][1] *= c_lo; o[i][2] *= c_hi; o[i][3] *= c_hi; }
        }
        const float ref_lo = m_lo == -INFINITY ? 0.f : m_lo, ref_hi = m_hi == -INFINITY ? 0.f : m_hi;
        uint32_t p[PF_KEYS / 16][4];
#pragma unroll
        for (int nt = 0; nt < PF_KEYS / 8; ++nt) {
            const float p0 = ex2(sc[nt][0] - ref_lo), p1 = ex2(sc[nt][1] - ref_lo);
            const float p2 = ex2(sc[nt][2] - ref_hi), p3 = ex2(sc[nt][3] - ref_hi);
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
static int log2_exact(int n) {               // -1: not a power of two
    if (n <= 0 || (n & (n - 1))) return -1;
    int l = 0;
    while ((1 << l) < n) ++l;
    return l;
}
static int merge(const float* scratch, const int* cu_q, void* out, int nH, int n_splits, int n_rows, int n_entries, int least, int most,
                 int rows, cudaStream_t stream) {
    const int z = rows < 1 ? 1 : rows > 65535 ? 65535 : rows;
    constexpr int G = 1024 / HD < 4 ? 1024 / HD : 4;
    if (n_splits > 4)
        NG_LAUNCH((attn_q8_merge_kernel<G>), dim3(nH, n_entries, z), G * HD, 0, stream, scratch, cu_q, (bf16*)out, nH, n_splits, n_rows, least, most);
    else
        NG_LAUNCH((attn_q8_merge_kernel<1>), dim3(nH, n_entries, z), HD, 0, stream, scratch, cu_q, (bf16*)out, nH, n_splits, n_rows, least, most);
    return ng_launch_status();
}

// scratch: n_rows * nH * n_splits * REC floats, 16-byte aligned (unused when n_splits == 1)
NG_EXPORT long long ng_attn_q8_scratch_floats(int n_rows, int nH, int n_splits) {
    return n_splits > 1 ? (long long)n_rows * nH * n_splits * REC : 0;
}

static bool cache_of(Cache& c, const void* k_pages, const void* v_pages, const float* ks, const float* vs, const int* table, int table_stride,
                     int nKV, int page_size, int block, int num_pages) {
    c = Cache{(const unsigned char*)k_pages, (const unsigned char*)v_pages, ks, vs, table, table_stride, num_pages, nKV, log2_exact(page_size),
              log2_exact(block)};
    return c.ps_log2 >= 3 && c.bl_log2 >= 3 && c.bl_log2 <= c.ps_log2 && nKV > 0 && table_stride > 0 && num_pages > 0 &&
           !(((uintptr_t)k_pages | (uintptr_t)v_pages) & 15);
}

NG_EXPORT int ng_attn_decode_q8(const void* q, const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                                const int* table, int table_stride, const int* cu_q, const int* ctx_before, void* out, float* scratch,
                                int n_rows, int n_entries, int nH, int nKV, int hd, int page_size, int block, int num_pages, int kind,
                                int window, float scale, int n_splits, int max_ctx, const float* slopes, cudaStream_t stream) {
    if (n_entries <= 0 || n_rows <= 0) return NG_OK;
    DcArgs a;
    if (hd != HD || nH <= 0 || !cache_of(a.c, k_pages, v_pages, k_scales, v_scales, table, table_stride, nKV, page_size, block, num_pages) ||
        nH % nKV || n_splits < 1 || n_splits > 65535 || n_entries > 65535 || (n_splits > 1 && (!scratch || ((uintptr_t)scratch & 15))) ||
        max_ctx < 0 || window < 0 || ((uintptr_t)q & 7) || (kind != NG_Q8_E4M3 && kind != NG_Q8_INT8))
        return NG_BAD_SIZE;
    const int G = nH / nKV;
    // a run: whole turns of the four warps; a window's first group may begin up to a group before it
    const long long span = (long long)(window > 0 && window < max_ctx ? window : max_ctx) + GROUP;
    const long long turn = DC_WARPS * GROUP, per = ((span + n_splits - 1) / n_splits + turn - 1) / turn * turn;
    a.q = (const bf16*)q; a.cu_q = cu_q; a.ctx_before = ctx_before; a.out = (bf16*)out; a.scratch = scratch; a.slopes = slopes;
    a.n_rows = n_rows; a.nH = nH; a.chunks = (G + 15) / 16; a.window = window; a.n_splits = n_splits; a.scale = scale;
    if (per * n_splits > 0x7fffffffll) return NG_BAD_SIZE;
    a.keys_per_split = (int)per;
    if ((long long)nKV * a.chunks > 0x7fffffffll) return NG_BAD_SIZE;
    const dim3 grid(nKV * a.chunks, n_entries, n_splits);
    const int smem = DC_WARPS * (G < 16 ? G : 16) * REC * (int)sizeof(float);
#define DC_GO(KIND)                                                                                                                   \
    do {                                                                                                                              \
        static std::atomic<unsigned long long> once{0};                                                                               \
        if (!ng_allow_smem(once, attn_decode_q8_kernel<KIND>, DC_WARPS * 16 * REC * (int)sizeof(float))) return NG_LAUNCH_FAILED;     \
        NG_LAUNCH((attn_decode_q8_kernel<KIND>), grid, DC_THREADS, smem, stream, a);                                                  \
    } while (0)
    if (kind == NG_Q8_E4M3) DC_GO(NG_Q8_E4M3);
    else DC_GO(NG_Q8_INT8);
    if (n_splits > 1) return merge(scratch, cu_q, out, nH, n_splits, n_rows, n_entries, 1, 1, 1, stream);
    return ng_launch_status();
}

NG_EXPORT int ng_attn_prefill_q8(const void* q, const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                                 const int* table, int table_stride, const int* cu_q, const int* ctx_before, void* out, float* scratch,
                                 int n_rows, int n_entries, int max_q, int nH, int nKV, int hd, int page_size, int block, int num_pages,
                                 int kind, int window, float scale, int skip_single, int n_splits, const float* slopes, cudaStream_t stream) {
    if (n_entries <= 0 || n_rows <= 0 || max_q <= 0) return NG_OK;
    PfArgs a;
    if (hd != HD || nH <= 0 || !cache_of(a.c, k_pages, v_pages, k_scales, v_scales, table, table_stride, nKV, page_size, block, num_pages) ||
        nH % nKV || n_splits < 1 || (long long)n_entries * n_splits > 65535 || (n_splits > 1 && (!scratch || ((uintptr_t)scratch & 15))) ||
        window < 0 || ((uintptr_t)q & 3) || ((uintptr_t)out & 3) || (kind != NG_Q8_E4M3 && kind != NG_Q8_INT8))
        return NG_BAD_SIZE;
    const long long rows = (long long)max_q * (nH / nKV), tiles = (rows + PF_ROWS - 1) / PF_ROWS;
    if (tiles > 65535) return NG_BAD_SIZE;
    a.q = (const bf16*)q; a.cu_q = cu_q; a.ctx_before = ctx_before; a.out = (bf16*)out; a.scratch = scratch; a.slopes = slopes;
    a.n_rows = n_rows; a.nH = nH; a.window = window; a.n_splits = n_splits; a.skip_single = skip_single; a.scale = scale;
    const dim3 grid(nKV, (unsigned)tiles, n_entries * n_splits);
#define PF_GO(KIND)                                                                                                  \
    do {                                                                                                             \
        static std::atomic<unsigned long long> once{0};                                                              \
        if (!ng_allow_smem(once, attn_prefill_q8_kernel<KIND>, (int)sizeof(PfSmem))) return NG_LAUNCH_FAILED;        \
        NG_LAUNCH((attn_prefill_q8_kernel<KIND>), grid, PF_THREADS, sizeof(PfSmem), stream, a);                      \
    } while (0)
    if (kind == NG_Q8_E4M3) PF_GO(NG_Q8_E4M3);
    else PF_GO(NG_Q8_INT8);
    if (n_splits > 1) return merge(scratch, cu_q, out, nH, n_splits, n_rows, n_entries, skip_single ? 2 : 1, 0x7fffffff, max_q, stream);
    return ng_launch_status();
}
