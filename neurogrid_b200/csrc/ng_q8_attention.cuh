// What the attention kernels over a cache in 8 bits share: the head size they are compiled for (-DNG_HEAD_DIM), the cache as their
// arguments have it, the records that runs of the keys leave and the kernel that merges them.
#pragma once
#include "ng_q8.cuh"

#ifndef NG_HEAD_DIM
#error "compile with -DNG_HEAD_DIM=<head size>"
#endif
#define HD NG_HEAD_DIM
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 in [16, 256]");
#define LOG2E 1.4426950408889634f
#define REC (HD + 4)            // floats of a run's record: reference point, sum, number of runs (single tokens), one unused, row in codes

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float q8_ex2(float x) {       // 2^x, 2 ulp; -inf -> 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// l 2^d + to, also where 2^d alone lies below the smallest normal number: a sum of 2^x over keys whose values have small scales is large (up to
// 2^100 a key) beside a reference point that contains the scales, and is still there when keys with the largest scales have moved that point by 2^200.
__device__ __forceinline__ float q8_add_scaled(float l, float d, float to) {
    const bool far = d < -125.f;
    const float c = q8_ex2(far ? 0.5f * d : d);
    return fmaf(far ? l * c : l, c, to);
}
// how far a run's reference point lies below the highest of several; runs that met only NaN have none, and keep their sums
__device__ __forceinline__ float q8_below(float ms, float m) { return m == -INFINITY ? 0.f : ms - m; }
// The denominator takes a key's weight 2^(z - m) divided by its scale, and the weight is lost below 2^-126.  m is the z of a key that counts 2^-(its log2
// scale) in the denominator, so what a lost key counts there is less than 2^-(126 - the distance of both scales' exponents) of it.  Keys
// whose scale's log2 is below Q8_LOW, and all once a scale above Q8_HIGH has moved m, are added by exponentials of their own: what others
// lose is below 2^-46.
#define Q8_LOW (-40)
#define Q8_HIGH 40
// The power of two that a row of q is divided by (its largest value becomes 1 to 2): exponent of the row's largest finite value.
__device__ __forceinline__ int q_exponent(float top) { return min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127); }
__device__ __forceinline__ float pow2_any(int e) { return q8_pow2(min(max(e, -126), 127)); }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

struct Cache {
    const unsigned char *k, *v;          // [pages, nKV, page, HD]
    const float *ks, *vs;                // [pages, nKV, page / block]
    const int* table;
    int table_stride, num_pages, nKV, ps_log2, bl_log2;
    int last_key;                        // the last position that a row of the table has a place for
};

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

// Which rows a block of a portion's launch has: tiles of `rows` (token, head) rows of each entry, entry by entry, an entry's from the last down (the
// blocks with the most keys start first); `index` counts them all.  Entries without rows, and single tokens where they are left out,
// have none, so that a launch beside many single tokens is not mostly blocks that find nothing to do (a portion of 512 tokens behind 2,000 beside 64
// single tokens 44 us; with a grid of entries x their longest's tiles 70, and cut into two runs 46 and, merged over that grid too, 356).  By
// a warp, 32 entries at a time.
struct RowTile { int e, first; };                                    // e < 0: behind the last tile
__device__ __forceinline__ RowTile row_tile(const int* cu_q, int n_entries, int n_rows, int group, int rows, bool skip_single, int index) {
    const int lane = threadIdx.x & 31;
    for (int e0 = 0; e0 < n_entries; e0 += 32) {
        int n = 0;
        if (e0 + lane < n_entries) {
            const int q0 = cu_q[e0 + lane], q1 = cu_q[e0 + lane + 1];
            if (q0 >= 0 && min(q1, n_rows) > q0 && !(skip_single && q1 - q0 == 1)) n = ((min(q1, n_rows) - q0) * group + rows - 1) / rows;
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const uint32_t in = __ballot_sync(0xffffffffu, index < upto);
        if (in) {
            const int l = __ffs(in) - 1;
            return RowTile{e0 + l, (__shfl_sync(0xffffffffu, upto, l) - 1 - index) * rows};
        }
        index -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return RowTile{-1, 0};
}
// the entry of a row (the last whose rows do not begin behind it), by a warp: 32 probes at a time; -1: none
__device__ __forceinline__ int entry_of_row(const int* cu_q, int n_entries, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n_entries;
    if (cu_q[0] > row || cu_q[n_entries] <= row) return -1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const int ahead = __popc(__ballot_sync(0xffffffffu, at < hi && cu_q[min(at, n_entries)] <= row));       // (lane 0's is)
        lo += (max(ahead, 1) - 1) * step;
        hi = min(lo + step, hi);
    }
    return lo;
}

// out[row, head] = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over the runs s.  A warp has a (row, head) (WIDE: all four warps of a block, every
// fourth run each, joined in order): lane s looks after run s's reference point and sum, then the lanes share the dimensions and walk the
// runs in ascending order.  SINGLE: rows are the entries' single tokens, with records by entry, of which the first says how many there are;
// else all rows of the entries that bring at least `least`.
#define MG_WARPS 4
constexpr int MG_EACH = (HD + 63) / 64;                              // pairs of dimensions a lane has
template <bool WIDE, bool SINGLE>
__global__ void __launch_bounds__(MG_WARPS * 32)
attn_q8_merge_kernel(const float* __restrict__ scratch, const int* __restrict__ cu_q, const int* __restrict__ ctx_before, int last_key,
                     bf16* __restrict__ out, int nH, int room, int n_rows, int n_entries, int least) {
    __shared__ float part_s[WIDE ? MG_WARPS : 1][HD + 2];
    ng_pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = WIDE ? blockIdx.x : blockIdx.x * MG_WARPS + warp;
    ng_pdl_wait();
    scratch = ng_after_wait(scratch);
    constexpr int STEP = WIDE ? MG_WARPS : 1;
    for (int i = blockIdx.y; i < (SINGLE ? n_entries : n_rows); i += gridDim.y) {
        const int e = SINGLE ? i : entry_of_row(cu_q, n_entries, i);
        if (e < 0) continue;
        const int q0 = cu_q[e], n = cu_q[e + 1] - q0, ctx = ctx_before[e], r = SINGLE ? q0 : i;
        if ((SINGLE ? n != 1 : n < least) || q0 < 0 || r >= n_rows || ctx < 0 || ctx > last_key || (!WIDE && head >= nH)) continue;      // (no records)
        const float* rec = scratch + ((size_t)i * nH + head) * room * REC;
        // (the first 32 runs' are asked for before it is known how many there are)
        const int s0 = lane * STEP + (WIDE ? warp : 0);
        float m0 = s0 < room ? rec[(size_t)s0 * REC] : -INFINITY, l0 = s0 < room ? rec[(size_t)s0 * REC + 1] : 0.f;
        int runs = room;
        if constexpr (SINGLE) {
            runs = (int)rec[2];
            if (runs <= 1) continue;
        }
        float m = -INFINITY, l = 0.f, acc[MG_EACH][2] = {};
        for (int b = 0; b < runs; b += 32 * STEP) {
            const int s1 = b + s0;
            float ms = m0, ls = l0;
            if (b > 0) {
                ms = s1 < runs ? rec[(size_t)s1 * REC] : -INFINITY;
                ls = s1 < runs ? rec[(size_t)s1 * REC + 1] : 0.f;
            }
            if (s1 >= runs) ms = -INFINITY, ls = 0.f;
            const float mb = fmaxf(m, ng_warp_max(ms)), c = q8_ex2(q8_below(m, mb)), f = q8_ex2(q8_below(ms, mb));
            l = q8_add_scaled(l, q8_below(m, mb), ng_warp_sum(q8_add_scaled(ls, q8_below(ms, mb), 0.f)));
            m = mb;
#pragma unroll
            for (int i = 0; i < MG_EACH; ++i) acc[i][0] *= c, acc[i][1] *= c;
            const uint32_t some = __ballot_sync(0xffffffffu, ls != 0.f);                               // (an empty run wrote no row)
            const int here = min(32, (runs - b - (WIDE ? warp : 0) + STEP - 1) / STEP);
#pragma unroll 4
            for (int k = 0; k < here; ++k) {
                const float fk = __shfl_sync(0xffffffffu, f, k);
                if (!(some >> k & 1)) continue;
                const float* row = rec + (size_t)(b + k * STEP + (WIDE ? warp : 0)) * REC + 4;
#pragma unroll
                for (int i = 0; i < MG_EACH; ++i) {
                    const int d = 2 * lane + 64 * i;
                    if (HD % 64 != 0 && d >= HD) continue;
                    const float2 x = *reinterpret_cast<const float2*>(row + d);
                    acc[i][0] = fmaf(x.x, fk, acc[i][0]);
                    acc[i][1] = fmaf(x.y, fk, acc[i][1]);
                }
            }
        }
        if constexpr (WIDE) {
            __syncthreads();                                         // the row before has been written
            if (lane == 0) part_s[warp][0] = m, part_s[warp][1] = l;
#pragma unroll
            for (int i = 0; i < MG_EACH; ++i) {
                const int d = 2 * lane + 64 * i;
                if (HD % 64 == 0 || d < HD) part_s[warp][2 + d] = acc[i][0], part_s[warp][3 + d] = acc[i][1];
            }
            __syncthreads();
            if (warp > 0) continue;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < MG_WARPS; ++w) top = fmaxf(top, part_s[w][0]);
            l = 0.f;
#pragma unroll
            for (int i = 0; i < MG_EACH; ++i) acc[i][0] = acc[i][1] = 0.f;
#pragma unroll
            for (int w = 0; w < MG_WARPS; ++w) {
                const float f = q8_ex2(q8_below(part_s[w][0], top));
                l = q8_add_scaled(part_s[w][1], q8_below(part_s[w][0], top), l);
#pragma unroll
                for (int i = 0; i < MG_EACH; ++i) {
                    const int d = 2 * lane + 64 * i;
                    if (HD % 64 == 0 || d < HD) acc[i][0] = fmaf(part_s[w][2 + d], f, acc[i][0]), acc[i][1] = fmaf(part_s[w][3 + d], f, acc[i][1]);
                }
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < MG_EACH; ++i) {
            const int d = 2 * lane + 64 * i;
            if (HD % 64 == 0 || d < HD)
                *reinterpret_cast<__nv_bfloat162*>(out + ((size_t)r * nH + head) * HD + d) = __floats2bfloat162_rn(acc[i][0] * inv, acc[i][1] * inv);
        }
    }
}

static int log2_exact(int n) {               // -1: not a power of two
    if (n <= 0 || (n & (n - 1))) return -1;
    int l = 0;
    while ((1 << l) < n) ++l;
    return l;
}
// The arguments of the attention entries, packed (a call through ctypes pays for every argument).
struct NgAttnQ8 {
    const void *q, *k_pages, *v_pages;
    const float *k_scales, *v_scales;
    const int *table, *cu_q, *ctx_before;
    void* out;
    float* scratch;
    const float* slopes;
    int* status;
    int table_stride, n_rows, n_entries, max_q, n_heads, n_kv, head_dim, page_size, block, num_pages, kind, window, skip_single, n_splits;
    float scale;
};
// What every entry refuses; fills in the cache.
static bool attn_q8_args(const NgAttnQ8& c, Cache& to) {
    to = Cache{(const unsigned char*)c.k_pages, (const unsigned char*)c.v_pages, c.k_scales, c.v_scales, c.table, c.table_stride, c.num_pages,
               c.n_kv, log2_exact(c.page_size), log2_exact(c.block), (int)((long long)c.table_stride * c.page_size - 1)};
    return c.head_dim == HD && c.n_heads > 0 && c.n_heads <= 1 << 20 && c.n_kv > 0 && c.n_heads % c.n_kv == 0 && to.ps_log2 >= 3 && to.bl_log2 >= 3 &&
           to.bl_log2 <= to.ps_log2 && c.table_stride > 0 && (long long)c.table_stride * c.page_size <= 1 << 30 && c.num_pages > 0 &&
           (long long)c.n_rows * c.n_heads <= 1 << 30 && (long long)c.n_kv * c.page_size * HD <= 0x7fffffff &&
           !(((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 15) && (c.kind == NG_Q8_E4M3 || c.kind == NG_Q8_INT8) && c.window >= 0 &&
           c.n_splits >= 1 && (c.n_splits == 1 || (c.scratch && !((uintptr_t)c.scratch & 15)));
}

// single: the entries' single tokens; else the rows of entries that bring at least `least`
static int q8_merge(const NgAttnQ8& c, const Cache& cache, bool single, int least, cudaStream_t stream) {
    const int count = single ? c.n_entries : c.n_rows;
    // A block a (row, head), or a warp: until the rows fill the GPU by themselves the wide form is the faster.  Heads of 64, with the attention in
    // front of it, wide / narrow, us: 1 row of 32 heads, 17 runs 8.3 / 11.9, 48 runs 15.5 / 24.6; 8 rows, 16 runs 11.2 / 11.9; 64 rows, 2 to
    // 16 runs 32.6 / 33.0 and 52.1 / 52.6; 256 rows, 8 runs 66.1 / 60.4; portions of 16 rows, 18 runs 34.7 / 38.4, 64 rows 41.2 / 45.6,
    // 128 rows, 9 runs 42.4 / 42.3, 512 rows, 2 runs 266 / 254
    const bool wide = (long long)count * c.n_heads <= 4096;
    const dim3 grid(wide ? c.n_heads : (c.n_heads + MG_WARPS - 1) / MG_WARPS, count < 65535 ? count : 65535);
#define MG_GO(WIDE, SINGLE)                                                                                                          \
    NG_LAUNCH((attn_q8_merge_kernel<WIDE, SINGLE>), grid, MG_WARPS * 32, 0, stream, c.scratch, c.cu_q, c.ctx_before, cache.last_key, \
              (bf16*)c.out, c.n_heads, c.n_splits, c.n_rows, c.n_entries, least)
    if (single && wide) MG_GO(true, true);
    else if (single) MG_GO(false, true);
    else if (wide) MG_GO(true, false);
    else MG_GO(false, false);
    return ng_launch_status();
}
// Row tiles that the portions' launch has to have room for: whole ones, and for each entry that may bring rows one that is not.
static long long q8_row_tiles(const NgAttnQ8& c, int rows) {
    const int group = c.n_heads / c.n_kv, least = c.skip_single ? 2 : 1;
    const long long whole = (long long)c.n_rows * group / rows, some = c.n_entries < c.n_rows / least ? c.n_entries : c.n_rows / least;
    const long long all = c.n_entries * (((long long)c.max_q * group + rows - 1) / rows);
    return all < whole + some ? all : whole + some;
}
