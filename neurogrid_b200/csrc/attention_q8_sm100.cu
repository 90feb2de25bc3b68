// Flash attention of prompt portions over a paged cache in 8 bits on the Blackwell tensor cores (head sizes 64 and 128, compiled with
// -DNG_HEAD_DIM).  The arithmetic is that of attention_q8.cu: codes as float16 operands, the keys' scales on the 32-bit scores,
// the values' scales in the exponents, the sum divided by them.
//
// A block owns two tiles of 128 rows of one (entry, KV head); a row is a (token, query head of the KV head), heads fastest, so that the heads
// which share keys share the key tiles that are fetched and turned into float16 for them, and both row tiles share them too.  Warps:
//   softmax     four for each stream; thread r of a stream owns row r of its row tile = TMEM lane r.  Heads of 64: a row tile has two
//               streams, which take the even and the odd key tiles, each with a reference point, a sum and an O of its own, joined at the end:
//               16 warps, four a scheduler, where eight waited for their own instructions most of the time.  Heads of 128 have one stream a row
//               tile (two O's of both do not fit TMEM).  Before the first key tile a stream brings its rows of q into shared memory
//   loaders (3) codes of the key tile after next from the pages into registers, while the tile before is stored as float16 in
//               the swizzled layout that the MMA reads (K row by row, V as it lies: [key][dim], MN-major)
//   issuer (1)  S = Q K^T and O += P V with tcgen05.mma, accumulators in TMEM, P taken from TMEM over S
// A row tile has two S buffers, for even and odd key tiles.  The tensor pipe runs the issuer's MMAs in order and a commit covers all
// before it, so "S of tile j + 2 is complete" also says that P V of tile j has read its P.
//
// Keys that no row of the block sees, and keys whose page is not there, are stored as zeros (their codes may be NaN).  The latter are hidden: the
// logarithm of their scale is minus infinity, and so is their z.  A NaN among the values of
// a key that some rows of the block see reaches the others of its tile as well (0 NaN), as it does in a plain product with masked weights.
// Denominators: a loader looks over the scales of the values as well.  If they lie so far apart that keys may have been lost to the denominator (Q8_LOW;
// this kernel's bound is FAR_SCALES), the rows' denominators are formed again at the end, key by key.  Exponentials of their own in such tiles, as in the
// other kernels, or the look at the scales in other warps, cost every cache 4 to 7 %: 2,048 tokens 41 -> 44 us, 512 behind 32,768 176 -> 184
// (so 42 and 180).  The same two over a cache of such values: 0.9 and 4.7 ms.
// Every mbarrier wait is bounded; a waiter that gives up sets a status bit and the block runs to its end.
//
// Bound by the softmax warps' instructions and by the handshakes of a tile (tensor pipe 28 %, exponential unit 56 %, issue slots 60 %
// busy): 0.93 us for 64 keys of 256 rows, and about 7 us for a block's start and end.  512 tokens behind 32,768 (24 / 8 heads of 64)
// 180 us = 577 TFLOP/s; 2,048 tokens, 32 / 8 heads of 64: 42 us; 6 requests of up to 611 tokens, 16 / 4 heads of 128, 65 us.  One row tile a block, two blocks an SM
// 221 us where this was 178; one stream a row tile 214; registers moved from loaders to softmax warps, exponentials of two streams in turn, two
// issuers, scores of 128 keys at once, 6 or 8 stages: no gain or slower.
#include <cstddef>
#include <type_traits>

#include "sm100_common.cuh"
#include "ng_q8_attention.cuh"

static_assert(HD == 64 || HD == 128, "head sizes 64 and 128");
#define BQ 128                       // rows of a row tile
#define BR (2 * BQ)                  // rows of a block
#define BK 64                        // keys of a tile
#define NB (HD / 64)                 // 64-wide blocks of a head
#define KV_STAGES 4
#define NG_STATUS_ATTN_TIMEOUT 16
#define STREAMS (HD == 64 ? 2 : 1)   // of a row tile
#define SOFTMAX_WARPS (8 * STREAMS)
#define Q8P_THREADS (32 * (SOFTMAX_WARPS + 4))
#define KV_WARPS 3
#define MIN_RUN 4                    // a run of keys is at least this many tiles
#define FAR_SCALES 100               // exponents' distance of scales up to which a key lost to the denominator counts less than 2^-26 of it
static_assert(BQ == BLOCK_W, "a row tile is the 128 rows of the MMA");

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two float32 values in one 64-bit register, and packed arithmetic on them (each half rounded as the scalar instruction rounds)
typedef unsigned long long u64;
__device__ __forceinline__ u64 pack2(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(u64 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ u64 ffma2(u64 a, u64 b, u64 c) {
    u64 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ u64 fadd2(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 32 consecutive float32 columns of this thread's TMEM lane, and 16 32-bit ones back
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
    float f[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
    tmem_st16(taddr, f);
}

struct Barriers {
    uint64_t q_full[2], kv_full[KV_STAGES], kv_empty[KV_STAGES], s_full[2][2], p_full[2][2], o_ready[2][2];          // [row tile][tile j & 1]
    uint64_t joined[2][4];                       // [row tile][warp]: the odd tiles' stream has left its reference point and sum
    uint64_t scales_seen;                        // `far` is known
};
struct Smem {
    uint16_t q[2][NB][BQ * 64];                  // K-major, 128-byte swizzle, a block for each 64 of the head
    uint16_t k[KV_STAGES][NB][BK * 64];
    uint16_t v[KV_STAGES][NB][BK * 64];
    float ks[KV_STAGES][8], vl[KV_STAGES][8], vi[KV_STAGES][8];       // of each 8 keys: K's scale, V's log2 and reciprocal
    Barriers b;
    float odd_m[BR], odd_l[BR], row_f[BR];       // row_f: what a row's raw products are multiplied by (base 2)
    uint32_t tmem_base, far;                     // far: scales of values lie more than FAR_SCALES apart
};

struct Params {
    Cache c;
    const bf16* q;
    bf16* out;
    const int *cu_q, *ctx_before;
    int* status;
    int n_rows, n_entries, nH, window, skip_single, n_splits;
    float scale;
    const float* slopes;
    float* scratch;
};

// half of a tile row's swizzled bytes: 16-byte chunk c (8 float16) of row r
__device__ __forceinline__ int sw128(int r, int c) { return (r >> 3) * 512 + (r & 7) * 64 + ((c ^ (r & 7)) << 3); }
// sum of 2^(x - top) over keys k0 .. k1 for row r of a row tile of q (float16, in shared memory), x = f * scale * (q . code) + slope (key - pos);
// eight keys at a time (they lie in one page and one block)
template <int KIND>
__device__ __noinline__ float denominator(const Cache& c, const int* trow, int kvh, const uint16_t* q, int r, float f, float slope, float top,
                                          int pos, int k0, int k1) {
    const int mask = (1 << c.ps_log2) - 1;
    float sum = 0.f;
#pragma unroll 1
    for (int key = k0 & ~7; key <= k1; key += 8) {
        const int i = key >> c.ps_log2, page = i < c.table_stride ? trow[i] : -1;
        if ((unsigned)page >= (unsigned)c.num_pages) continue;
        const long long slab = (long long)page * c.nKV + kvh;
        const unsigned char* codes = c.k + ((slab << c.ps_log2) + (key & mask)) * HD;
        const float fk = f * c.ks[(slab << (c.ps_log2 - c.bl_log2)) + ((key & mask) >> c.bl_log2)];
        float raw[8] = {};
#pragma unroll 1
        for (int ch = 0; ch < HD / 8; ++ch) {                  // eight dimensions
            uint32_t w[8][2];
#pragma unroll
            for (int n = 0; n < 8; ++n) ld_codes<8>(w[n], codes + n * HD + ch * 8);
            const uint4 x = *reinterpret_cast<const uint4*>(q + ch / 8 * (BQ * 64) + sw128(r, ch % 8));
            const uint32_t qs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t h[2];
                    q8_to_half<KIND>(w[n][j], h[0], h[1]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&qs[2 * j + u])), b = __half22float2(*reinterpret_cast<const __half2*>(&h[u]));
                        raw[n] = fmaf(a.x, b.x, fmaf(a.y, b.y, raw[n]));
                    }
                }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n)
            if (key + n >= k0 && key + n <= k1) sum += q8_ex2(fmaf(raw[n], fk, slope * (float)(key + n - pos)) - top);
    }
    return sum;
}
// kind::f16, float16 operands: as make_idesc without its bfloat16 bits
__host__ __device__ constexpr uint32_t idesc_f16(int n, int b_mn) { return make_idesc(n, b_mn) & ~((1u << 7) | (1u << 10)); }

template <int KIND>
__global__ void __launch_bounds__(Q8P_THREADS, 1)
attn_prefill_q8_sm100_kernel(const __grid_constant__ Params p) {
    extern __shared__ unsigned char smem_raw[];
    // (an offset, not a rounded address: the compiler then knows that what it points to is shared memory)
    Smem* sm = reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    const bool leader = elected != 0;
    const int split = blockIdx.z, kvh = blockIdx.x, G = p.nH / p.c.nKV;
    const RowTile mine = row_tile(p.cu_q, p.n_entries, p.n_rows, G, BR, p.skip_single, blockIdx.y);
    const int e = max(mine.e, 0), r0 = mine.first;
    const int q0 = p.cu_q[e], qlen = min(p.cu_q[e + 1], p.n_rows) - q0, ctx = p.ctx_before[e];
    if (mine.e < 0 || ctx < 0 || ctx > p.c.last_key) {
        ng_pdl_wait();                                         // (a launch none of whose blocks waited would end before the one before it)
        return;
    }
    // A row of the block is of token tb + tr; n rows behind the first one of token tb: (n + 1/2) / G in float32 is exact for n < 2^21
    const int tb = r0 / G, hb = r0 - tb * G;
    const float per_head = 1.f / (float)G;
    auto row_at = [&](int row) {                               // of the block; the row's place in q and out, in rows of heads
        const int n = hb + row, tr = (int)(((float)n + 0.5f) * per_head);
        return (size_t)(q0 + tb + tr) * p.nH + kvh * G + n - tr * G;
    };
    const int rows_here = min(BR, qlen * G - r0), rows_0 = min(BQ, rows_here), rows_1 = max(0, rows_here - BQ);
    const int first = ctx + r0 / G, last = ctx + (r0 + rows_here - 1) / G;          // positions
    const int key_lo = p.window > 0 ? max(0, first - p.window + 1) : 0, kv_end = last + 1;
    int tile0 = key_lo / BK, tile1 = last / BK;                // inclusive
    if (p.n_splits > 1) {
        const int per = max(MIN_RUN, (tile1 - tile0 + p.n_splits) / p.n_splits);
        tile0 += split * per;
        tile1 = min(tile1, tile0 + per - 1);
    }
    // key tiles of each row tile: the first one's rows see less
    const int n_0 = min(tile1, (ctx + (r0 + rows_0 - 1) / G) / BK) - tile0 + 1, n_1 = rows_1 > 0 ? tile1 - tile0 + 1 : 0;
    const int n_tiles = max(n_0, n_1);
    if (n_tiles <= 0) {                                        // an empty run: records that the merge passes over
        ng_pdl_wait();
        if (threadIdx.x < rows_here) {
            float* rec = p.scratch + (row_at(threadIdx.x) * p.n_splits + split) * REC;
            rec[0] = -INFINITY;
            rec[1] = 0.f;
        }
        return;
    }
    if (threadIdx.x < sizeof(Barriers) / 8) {                  // a thread a barrier
        const int i = threadIdx.x;
        const bool kv = i >= offsetof(Barriers, kv_full) / 8 && i < offsetof(Barriers, kv_empty) / 8, pf = i >= offsetof(Barriers, p_full) / 8 && i < offsetof(Barriers, o_ready) / 8;
        mbar_init(reinterpret_cast<uint64_t*>(&sm->b) + i, i < 2 ? 4 * STREAMS : kv ? KV_WARPS : pf ? 4 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Loaders: the page numbers of the first tiles (the batch description: no kernel of this step writes it)
    constexpr int UNITS = (8 + KV_WARPS - 1) / KV_WARPS, DEPTH = 2;
    const int loader = __shfl_sync(0xffffffffu, warp - SOFTMAX_WARPS, 0);
    struct Pages { int unit[UNITS], mine; };                   // of a tile to ask for, as the table has them; mine: lane u's, unit u's (the scales)
    auto page_of = [&](int key) {                              // (not looked at before the tile is asked for: the load would be waited for here)
        const int i = key >> p.c.ps_log2;
        return key + 7 >= key_lo && key < kv_end && i < p.c.table_stride ? p.c.table[(size_t)e * p.c.table_stride + i] : -1;
    };
    auto pages = [&](int tile) {
        Pages to;
#pragma unroll
        for (int n = 0; n < UNITS; ++n) to.unit[n] = loader + KV_WARPS * n < 8 ? page_of(tile * BK + 8 * (loader + KV_WARPS * n)) : -1;
        to.mine = loader == KV_WARPS - 1 && lane < 8 ? page_of(tile * BK + 8 * lane) : -1;
        return to;
    };
    Pages page0{}, page1{};
    if (loader >= 0 && loader < KV_WARPS) page0 = pages(tile0), page1 = pages(tile0 + 1);
    ng_pdl_wait();                                             // q and the pages are this step's data
    // All of the SM's tensor memory: asked for behind the wait, and the next kernel let in behind the allocation.  A block of a tcgen05 product of few
    // rows fits on the SM beside this one (its 4,096 registers and 110 KB are what is left): had it tensor memory before this block did, this
    // block would wait for it, and it for this kernel (or, in front of this kernel, this block for it and it for the tensor memory).
    if (warp == SOFTMAX_WARPS + KV_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_u32(&sm->tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    ng_pdl_trigger();
    const uint32_t tmem = sm->tmem_base;                       // S of row tile t, tile j: 128 t + 64 (j & 1); O: tm_o(t, j)
    auto tm_o = [&](int t, int j) { return tmem + 256 + HD * (STREAMS == 2 ? 2 * t + (j & 1) : t); };
    bool ok = true;

    if (warp >= SOFTMAX_WARPS && warp < SOFTMAX_WARPS + KV_WARPS) {
        // ------------------------------------------------------------------ keys and values
        // A unit is eight keys (they lie in one page and one block) of K and of V: UNIT_LOADS requests of 16 bytes a lane each.  A warp has
        // every third unit; page numbers are asked for a tile before the codes, the codes DEPTH tiles before they are stored.
        constexpr int UNIT_LOADS = HD / 64;
        const int w = loader, mask = (1 << p.c.ps_log2) - 1;
        const long long page_bytes = (long long)(p.c.nKV << p.c.ps_log2) * HD, head_at = (long long)(kvh << p.c.ps_log2) * HD + lane * 16;
        const unsigned char *k_pages = p.c.k + head_at, *v_pages = p.c.v + head_at;
        uint32_t k[DEPTH][UNITS][UNIT_LOADS][4], v[DEPTH][UNITS][UNIT_LOADS][4];
        float ks[DEPTH], vs[DEPTH];                            // (vs: -1 for a unit that has no page)
        float low = INFINITY, high = 0.f;                      // the last loader's lanes: scales of values so far
        // (a page that is not there: page 0 is read, and the unit's keys become zeros when they are stored)
        bool bad[DEPTH][UNITS];
        auto load = [&](int d, int tile, const Pages& page) {
#pragma unroll
            for (int n = 0; n < UNITS; ++n) {
                bad[d][n] = (unsigned)page.unit[n] >= (unsigned)p.c.num_pages;
                const long long at = (long long)(bad[d][n] ? 0 : page.unit[n]) * page_bytes + (tile * BK + 8 * (w + KV_WARPS * n) & mask) * HD;
#pragma unroll
                for (int i = 0; i < UNIT_LOADS; ++i) {
                    ld_codes<16>(k[d][n][i], k_pages + at + i * 512);
                    ld_codes<16>(v[d][n][i], v_pages + at + i * 512);
                }
            }
            ks[d] = 1.f;
            vs[d] = -1.f;
            if ((unsigned)page.mine < (unsigned)p.c.num_pages) {
                const long long sc = ((long long)page.mine * p.c.nKV + kvh << (p.c.ps_log2 - p.c.bl_log2)) + ((tile * BK + 8 * lane & mask) >> p.c.bl_log2);
                ld_codes<4>(reinterpret_cast<uint32_t*>(&ks[d]), reinterpret_cast<const unsigned char*>(p.c.ks + sc));
                ld_codes<4>(reinterpret_cast<uint32_t*>(&vs[d]), reinterpret_cast<const unsigned char*>(p.c.vs + sc));
            }
        };
        auto put = [](uint16_t* tile, int row, int c, const uint32_t (&x)[4]) {          // 16 codes: chunks c and c + 1 of the row
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) q8_to_half<KIND>(x[i], h[2 * i], h[2 * i + 1]);
            *reinterpret_cast<uint4*>(tile + sw128(row, c)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(tile + sw128(row, c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
        };
        static_assert(DEPTH == 2, "two tiles are asked for here");
        load(0, tile0, page0);
        load(1, tile0 + 1, page1);
        page0 = pages(tile0 + DEPTH);
        for (int j0 = 0; j0 < n_tiles && ok; j0 += DEPTH)
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int j = j0 + d, s = j % KV_STAGES;
                if (j >= n_tiles || !ok) break;
                ok = __all_sync(0xffffffffu, mbar_wait(&sm->b.kv_empty[s], ((j / KV_STAGES) & 1) ^ 1));
                if (!ok) break;
#pragma unroll
                for (int n = 0; n < UNITS; ++n)
                    if (w + KV_WARPS * n < 8) {
                        const int key0 = (tile0 + j) * BK + 8 * (w + KV_WARPS * n);
                        if (bad[d][n] || key0 < key_lo || key0 + 8 > kv_end)         // keys that no row sees: zeros
#pragma unroll
                            for (int i = 0; i < UNIT_LOADS; ++i) {
                                const int key = key0 + (i * 512 + lane * 16) / HD;
                                if (bad[d][n] || key < key_lo || key >= kv_end)
#pragma unroll
                                    for (int x = 0; x < 4; ++x) k[d][n][i][x] = v[d][n][i][x] = 0u;
                            }
#pragma unroll
                        for (int i = 0; i < UNIT_LOADS; ++i) {
                            const int o = i * 512 + lane * 16, row = 8 * (w + KV_WARPS * n) + o / HD, c = o % HD / 8;
                            put(sm->k[s][c / 8], row, c % 8, k[d][n][i]);
                            put(sm->v[s][c / 8], row, c % 8, v[d][n][i]);
                        }
                    }
                if (w == KV_WARPS - 1 && lane < 8) {
                    sm->ks[s][lane] = ks[d];
                    sm->vl[s][lane] = vs[d] < 0.f ? -INFINITY : q8_log2(vs[d]);
                    low = fminf(low, vs[d] < 0.f ? INFINITY : vs[d]), high = fmaxf(high, vs[d]);
                    sm->vi[s][lane] = q8_recip(vs[d]);         // (of a unit without a page: 1, times weights of 0)
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm->b.kv_full[s]);
                load(d, tile0 + j + DEPTH, page0);             // (behind the last tile: zeros, from no page)
                page0 = pages(tile0 + j + DEPTH + 1);
            }
        if (w == KV_WARPS - 1) {
            const bool far = __any_sync(0xffffffffu, q8_log2(ng_warp_max(high)) - q8_log2(low) > FAR_SCALES);
            if (lane == 0) {
                sm->far = far;
                mbar_arrive(&sm->b.scales_seen);
            }
        }
        if (!ok && lane == 0) atomicOr(p.status, NG_STATUS_ATTN_TIMEOUT);
    } else if (warp == SOFTMAX_WARPS + KV_WARPS) {
        // ------------------------------------------------------------------ MMA issuer: all lanes run the loop, one issues
        constexpr uint32_t idesc_s = idesc_f16(BK, 0), idesc_o = idesc_f16(64, 1);
        for (int t = 0; t < 2 && ok; ++t)
            if ((t ? n_1 : n_0) > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sm->b.q_full[t], 0));
        // descriptors of the first stage; addresses are in units of 16 bytes, and so are the distances added to them
        const uint64_t q_desc = make_desc_sw128(sm->q[0][0]), k_desc = make_desc_sw128(sm->k[0][0]), v_desc = make_desc_sw128_mn(sm->v[0][0]);
        constexpr uint64_t Q_TILE = sizeof(sm->q[0]) / 16, Q_BLOCK = sizeof(sm->q[0][0]) / 16, KV_STAGE = sizeof(sm->k[0]) / 16, KV_BLOCK = sizeof(sm->k[0][0]) / 16;
        auto issue_s = [&](int t, int j) {                     // S = Q K_j^T into buffer j & 1 of row tile t
            const int s = j % KV_STAGES;
            if (!__all_sync(0xffffffffu, mbar_wait(&sm->b.kv_full[s], (j / KV_STAGES) & 1))) { ok = false; return; }
            tcgen05_fence_after();
            if (leader) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint64_t dq = q_desc + t * Q_TILE + b * Q_BLOCK, dk = k_desc + s * KV_STAGE + b * KV_BLOCK;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tcgen05_mma_f16(tmem + 128 * t + 64 * (j & 1), dq + (uint64_t)(2 * k), dk + (uint64_t)(2 * k), idesc_s, b > 0 || k > 0);
                }
                tcgen05_commit(&sm->b.s_full[t][j & 1]);
            }
            __syncwarp();
        };
        for (int j = 0; j < 2; ++j)
            for (int t = 0; t < 2; ++t)
                if (ok && j < (t ? n_1 : n_0)) issue_s(t, j);
        for (int j = 0; j < n_tiles && ok; ++j) {
            const int s = j % KV_STAGES;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int n = t ? n_1 : n_0;
                if (!ok) break;
                if (j < n) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sm->b.p_full[t][j & 1], (j >> 1) & 1));          // P_j in tensor memory, O rescaled
                    if (!ok) break;
                    tcgen05_fence_after();
                    if (leader) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const uint64_t dv = v_desc + s * KV_STAGE + b * KV_BLOCK;
#pragma unroll
                            for (int k = 0; k < BK / 16; ++k)  // 16 keys an MMA: 8 columns of P, 2,048 bytes of V
                                tcgen05_mma_f16_ts(tm_o(t, j) + 64 * b, tmem + 128 * t + 64 * (j & 1) + 8 * k, dv + (uint64_t)(128 * k),
                                                   idesc_o, j >= STREAMS || k > 0);
                        }
                        tcgen05_commit(&sm->b.o_ready[t][j & 1]);                // O holds tiles 0..j
                    }
                }
                if (t == 1 && leader) tcgen05_commit(&sm->b.kv_empty[s]);        // K_j and V_j may be overwritten
                __syncwarp();
                if (j + 2 < n) issue_s(t, j + 2);
            }
        }
        if (!ok && leader) atomicOr(p.status, NG_STATUS_ATTN_TIMEOUT);
    } else {
        // ------------------------------------------------------------------ softmax: thread = row
        const int t = warp / (4 * STREAMS), odd = STREAMS == 2 ? warp >> 2 & 1 : 0, r = threadIdx.x & (BQ - 1);
        const int n_mine = t ? n_1 : n_0, rows_mine = t ? rows_1 : rows_0;
        const int rr = r0 + BQ * t + min(r, max(rows_mine, 1) - 1);        // rows past the last mirror it
        const int token = rr / G, head = kvh * G + rr - token * G, pos = ctx + token;
        const int pos_first = ctx + (r0 + BQ * t) / G, pos_last = ctx + (r0 + BQ * t + max(rows_mine, 1) - 1) / G;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        float f = 0.f;
        if (n_mine > 0) {
            // The warp's rows of q (of two streams, each brings 16 of the 32), each divided by a power of two, as float16: eight lanes a row, so
            // that a request is whole lines, all in flight.  (A thread a row: 4 us at the start of every block, heads of 128 7 us.)
            constexpr int ROWS = 4, MINE = 32 / STREAMS;
            const bf16* q = ng_after_wait(p.q);
            const int c = lane & 7, at = 32 * (warp & 3) + MINE * odd + (lane >> 3);     // 16-byte chunk of 64 dimensions; row of the row tile
#pragma unroll 4
            for (int i = 0; i < MINE; i += ROWS) {             // (rows past the last read that one)
                const bf16* from = q + row_at(BQ * t + min(at + i, rows_mine - 1)) * HD + 8 * c;
#pragma unroll
                for (int n = 0; n < NB; ++n)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(sm->q[t][n] + sw128(at + i, c))), "l"(from + 64 * n) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");   // (a lane reads what it asked for itself)
#pragma unroll 2
            for (int i = 0; i < MINE; i += ROWS) {
                uint4 w[NB];
                float top = 0.f;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    w[n] = *reinterpret_cast<const uint4*>(sm->q[t][n] + sw128(at + i, c));
                    const uint32_t x[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a = fabsf(__uint_as_float(x[j] << 16)), b = fabsf(__uint_as_float(x[j] & 0xffff0000u));
                        if (a < INFINITY) top = fmaxf(top, a);
                        if (b < INFINITY) top = fmaxf(top, b);
                    }
                }
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const int ex = q_exponent(top);
                const float div = pow2_any(-ex);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const uint32_t x[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
                    uint32_t h[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[j] = pack_f16(__uint_as_float(x[j] << 16) * div, __uint_as_float(x[j] & 0xffff0000u) * div);
                    *reinterpret_cast<uint4*>(sm->q[t][n] + sw128(at + i, c)) = make_uint4(h[0], h[1], h[2], h[3]);
                }
                if (c == 0) sm->row_f[BQ * t + at + i] = p.scale * LOG2E * pow2_any(ex);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm->b.q_full[t]);
            if constexpr (STREAMS == 2) asm volatile("bar.sync %0, 64;" :: "r"(1 + 4 * t + (warp & 3)) : "memory");        // the two warps of these rows
            f = sm->row_f[BQ * t + r];
        }
        // m is the reference point of the exponentials; it moves to the first tile's maximum and then follows lazily: only when a tile exceeds
        // it by more than 2^8 is O in TMEM rescaled (which has to wait for the product before).
        float m = 0.f, l = 0.f;
        bool seen = false;
        const float slope = p.slopes ? p.slopes[head] * LOG2E : 0.f;
        for (int j = odd; j < n_mine && ok; j += STREAMS) {
            const int s = j % KV_STAGES, key0 = (tile0 + j) * BK;
            ok = mbar_wait(&sm->b.kv_full[s], (j / KV_STAGES) & 1) && mbar_wait(&sm->b.s_full[t][j & 1], (j >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tcgen05_fence_after();
            const uint32_t ts = tmem + 128 * t + 64 * (j & 1) + lane_base;
            float corr = 1.f;
            // z = sc fk + lg + slope (key - pos), 32 keys of the row at a time; where no key is hidden the largest z of each eight keys has the
            // largest sc (f and the scales are positive), or with a bias the largest sc fk + slope i.  The first pass finds the maximum, the
            // second the weights: the last 32 scores are still there, the first are read again.
            auto weigh = [&](auto kind) {
                constexpr int MODE = decltype(kind)::value;                // 0: plain, 1: a bias, 2: hidden keys (and a bias, if only of 0)
                const float far = slope * (float)(key0 - pos);
                const int rel = pos - key0, out_of = p.window > 0 ? rel - p.window : -1;
                uint32_t vis[2];                                           // a bit for each key that the row sees: out_of < key - key0 <= rel
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int n = min(max(rel + 1 - 32 * h, 0), 32), n0 = min(max(out_of + 1 - 32 * h, 0), 32);
                    vis[h] = (uint32_t)((1ull << n) - (1ull << min(n0, n)));
                }
                float sc[32];
                auto formed = [&](int b, float ks) {                       // the eight scores at 8 b become z less lg and far (1, 2)
                    if constexpr (MODE >= 1) {
                        const float fk = f * ks;
                        const u64 fk2 = pack2(fk, fk);
#pragma unroll
                        for (int i = 0; i < 8; i += 2)
                            unpack2(ffma2(pack2(sc[8 * (b & 3) + i], sc[8 * (b & 3) + i + 1]), fk2, pack2(slope * i, slope * (i + 1))),
                                    sc[8 * (b & 3) + i], sc[8 * (b & 3) + i + 1]);
                        if constexpr (MODE == 2)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (!(vis[b >> 2] >> (8 * (b & 3) + i) & 1)) sc[8 * (b & 3) + i] = -INFINITY;
                    }
                };
                float mx = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tmem_ld32(ts + 32 * h, sc);
                    const float4 k4 = *reinterpret_cast<const float4*>(&sm->ks[s][4 * h]), v4 = *reinterpret_cast<const float4*>(&sm->vl[s][4 * h]);
                    const float ks[4] = {k4.x, k4.y, k4.z, k4.w}, vl[4] = {v4.x, v4.y, v4.z, v4.w};
                    float mz[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        formed(4 * h + u, ks[u]);
                        const float* x = sc + 8 * u;
                        const float y = fmaxf(fmax3(fmax3(x[0], x[1], x[2]), fmax3(x[3], x[4], x[5]), x[6]), x[7]);
                        mz[u] = MODE == 0 ? fmaf(y, f * ks[u], vl[u]) : y + (vl[u] + fmaf(8.f * slope, (float)(4 * h + u), far));
                    }
                    mx = fmax3(mx, fmaxf(mz[0], mz[1]), fmaxf(mz[2], mz[3]));
                }
                if (mx > m + 8.f || (!seen && mx > -INFINITY)) {           // move the reference point
                    corr = seen ? q8_ex2(m - mx) : 0.f;        // (sums that this loses: FAR_SCALES)
                    seen = true;
                    m = mx;
                    l *= corr;
                }
                uint32_t late[16];
#pragma unroll
                for (int h = 1; h >= 0; --h) {
                    if (h == 0) {
                        tmem_ld32(ts, sc);
                        tmem_st16u(ts + 16, late);                         // (over scores that have just been read again)
                    }
                    uint32_t pk[16];
                    const float4 k4 = *reinterpret_cast<const float4*>(&sm->ks[s][4 * h]), v4 = *reinterpret_cast<const float4*>(&sm->vl[s][4 * h]);
                    const float4 i4 = *reinterpret_cast<const float4*>(&sm->vi[s][4 * h]);
                    const float ks[4] = {k4.x, k4.y, k4.z, k4.w}, vl[4] = {v4.x, v4.y, v4.z, v4.w}, vi[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (h == 0) formed(u, ks[u]);
                        const float fk = f * ks[u], lg = (MODE == 0 ? vl[u] : vl[u] + fmaf(8.f * slope, (float)(4 * h + u), far)) - m;
                        const u64 fk2 = pack2(fk, fk), lg2 = pack2(lg, lg);
                        u64 sum2 = pack2(0.f, 0.f);
#pragma unroll
                        for (int i = 8 * u; i < 8 * u + 8; i += 2) {
                            float x, y;
                            unpack2(MODE == 0 ? ffma2(pack2(sc[i], sc[i + 1]), fk2, lg2) : fadd2(pack2(sc[i], sc[i + 1]), lg2), x, y);
                            x = q8_ex2(x), y = q8_ex2(y);
                            sum2 = fadd2(sum2, pack2(x, y));
                            pk[i / 2] = pack_f16(x, y);
                        }
                        float x, y;
                        unpack2(sum2, x, y);
                        l = fmaf(x + y, vi[u], l);
                    }
                    if (h == 0) tmem_st16u(ts, pk);
                    else
#pragma unroll
                        for (int i = 0; i < 16; ++i) late[i] = pk[i];
                }
            };
            // only tiles that cross a row's diagonal or the window's edge have hidden keys
            if (!(key0 + BK - 1 <= pos_first && (p.window <= 0 || key0 > pos_last - p.window))) weigh(std::integral_constant<int, 2>{});
            else if (p.slopes) weigh(std::integral_constant<int, 1>{});
            else weigh(std::integral_constant<int, 0>{});
            if (j >= STREAMS && __any_sync(0xffffffffu, corr != 1.f)) {    // rescale this warp's rows of O
                ok = mbar_wait(&sm->b.o_ready[t][(j - STREAMS) & 1], ((j - STREAMS) >> 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tcgen05_fence_after();
#pragma unroll
                for (int c = 0; c < HD; c += 16) {
                    float x[16];
                    tmem_ld16(tm_o(t, j) + lane_base + c, x);
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] *= corr;
                    tmem_st16(tm_o(t, j) + lane_base + c, x);
                }
            }
            // P lies over this row's S (whose last other reader, the product of tile j - 2, is complete with S_j)
            tmem_st_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm->b.p_full[t][j & 1]);
        }
        // what the odd tiles' stream found goes to the even tiles', which writes the rows
        const int last_j = n_mine - 1 - (STREAMS == 2 && (n_mine - 1 & 1) != odd ? 1 : 0);             // the stream's last tile (< 0: none)
        if (ok && n_mine > 0 && last_j >= 0) {
            ok = mbar_wait(&sm->b.o_ready[t][last_j & 1], (last_j >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!odd && ok && n_mine > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sm->b.scales_seen, 0));
        float m_odd = -INFINITY, l_odd = 0.f;
        if (STREAMS == 2 && n_mine > 1 && ok) {
            if (odd) {
                tcgen05_fence_before();
                sm->odd_m[BQ * t + r] = seen ? m : -INFINITY;
                sm->odd_l[BQ * t + r] = l;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm->b.joined[t][warp & 3]);
            } else {
                ok = __all_sync(0xffffffffu, mbar_wait(&sm->b.joined[t][warp & 3], 0));
                m_odd = sm->odd_m[BQ * t + r];
                l_odd = sm->odd_l[BQ * t + r];
            }
        }
        if (!ok) {
            if (lane == 0) atomicOr(p.status, NG_STATUS_ATTN_TIMEOUT);
        } else if (!odd) {
            float* rec = p.scratch + (row_at(BQ * t + r) * p.n_splits + split) * REC;
            const bool two = STREAMS == 2 && n_mine > 1, live = r < rows_mine;
            const float m_even = seen ? m : -INFINITY, top = fmaxf(m_even, m_odd);
            // (a stream that met only NaN has no reference point and keeps its sums)
            float a = q8_ex2(q8_below(m_even, top)), b = q8_ex2(q8_below(m_odd, top));
            l = fmaf(l, a, l_odd * b);
            if (n_mine <= 0) l = 0.f;
            else if (sm->far && live && top > -INFINITY) {
                l = denominator<KIND>(p.c, p.c.table + (size_t)e * p.c.table_stride, kvh, sm->q[t][0], r, f, slope, top, pos,
                                      max(tile0 * BK, p.window > 0 ? pos - p.window + 1 : 0), min((tile0 + n_mine) * BK - 1, pos));
            }
            if (p.n_splits > 1 && live) rec[0] = n_mine > 0 ? top : -INFINITY, rec[1] = l;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (p.n_splits == 1) a *= inv, b *= inv;
            if (n_mine > 0) {
                tcgen05_fence_after();
                constexpr int CH = STREAMS == 1 ? 32 : 16;     // dimensions at a time
#pragma unroll 1
                for (int c = 0; c < HD; c += CH) {
                    float x[CH], y[CH];
                    if constexpr (STREAMS == 1) tmem_ld32(tm_o(t, 0) + lane_base + c, x);
                    else tmem_ld16(tm_o(t, 0) + lane_base + c, x);
                    if constexpr (STREAMS == 2)
                        if (two) tmem_ld16(tm_o(t, 1) + lane_base + c, y);
#pragma unroll
                    for (int i = 0; i < CH; ++i) x[i] = two ? fmaf(x[i], a, y[i] * b) : x[i] * a;
                    if (p.n_splits > 1) {
                        if (live)
#pragma unroll
                            for (int i = 0; i < CH; i += 4) *reinterpret_cast<float4*>(rec + 4 + c + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                        continue;
                    }
#pragma unroll
                    for (int i = 0; i < CH; i += 8) {          // over the rows of q, which no product reads any more
                        uint32_t w[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(x[i + 2 * u], x[i + 2 * u + 1]);
                            w[u] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        *reinterpret_cast<uint4*>(sm->q[t][(c + i) / 64] + sw128(r, (c + i) / 8 % 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                if (p.n_splits == 1) {                         // whole lines again
                    __syncwarp();
                    constexpr int LANES = HD / 8, ROWS = 32 / LANES;
                    const int c = lane % LANES, at = 32 * (warp & 3) + lane / LANES;
#pragma unroll 4
                    for (int i = 0; i < 32; i += ROWS)
                        if (at + i < rows_mine)
                            *reinterpret_cast<uint4*>(p.out + row_at(BQ * t + at + i) * HD + 8 * c) =
                                *reinterpret_cast<const uint4*>(sm->q[t][c / 8] + sw128(at + i, c % 8));
                }
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == SOFTMAX_WARPS + KV_WARPS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
}

// scratch (n_splits > 1): n_rows * n_heads * n_splits * REC floats, 16-byte aligned
NG_EXPORT int ng_attn_prefill_q8_sm100(const NgAttnQ8* call, cudaStream_t stream) {
    const NgAttnQ8& c = *call;
    const int kind = c.kind;
    if (c.n_entries <= 0 || c.n_rows <= 0 || c.max_q <= 0) return NG_OK;
    Params p;
    if (!attn_q8_args(c, p.c) || c.n_splits > 65535 || !(c.scale > 0.f) || !c.status ||
        (((uintptr_t)c.q | (uintptr_t)c.out) & 15))
        return NG_BAD_SIZE;
    const long long tiles = q8_row_tiles(c, BR);
    if (tiles > 65535) return NG_BAD_SIZE;
    if (tiles <= 0) return NG_OK;                              // (one row, and single tokens are left out)
    p.q = (const bf16*)c.q; p.out = (bf16*)c.out; p.cu_q = c.cu_q; p.ctx_before = c.ctx_before; p.status = c.status; p.n_rows = c.n_rows; p.n_entries = c.n_entries;
    p.nH = c.n_heads; p.window = c.window; p.skip_single = c.skip_single; p.n_splits = c.n_splits; p.scale = c.scale; p.slopes = c.slopes;
    p.scratch = c.scratch;
    const dim3 grid(c.n_kv, (unsigned)tiles, c.n_splits);
    constexpr int smem = (int)sizeof(Smem) + 1024;
#define Q8P_GO(KIND)                                                                                                     \
    do {                                                                                                                 \
        static std::atomic<unsigned long long> once{0};                                                                  \
        if (!ng_allow_smem(once, attn_prefill_q8_sm100_kernel<KIND>, smem)) return NG_LAUNCH_FAILED;                     \
        NG_LAUNCH((attn_prefill_q8_sm100_kernel<KIND>), grid, Q8P_THREADS, smem, stream, p);                             \
    } while (0)
    if (kind == NG_Q8_E4M3) Q8P_GO(NG_Q8_E4M3);
    else Q8P_GO(NG_Q8_INT8);
    if (c.n_splits > 1) return q8_merge(c, p.c, false, c.skip_single ? 2 : 1, stream);
    return ng_launch_status();
}
