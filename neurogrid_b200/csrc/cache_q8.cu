// A paged cache of keys and values in 8 bits: its writer, and the copying of pages.
#include <cstdlib>
#include <type_traits>

#include "ng_q8.cuh"

// ===================================================================================== write
// New keys and values of a ragged batch into their pages, in codes with a scale for each block of tokens and KV head (ng_q8.cuh).
//
// A block of a request may fill over many steps, so its scale is found from what is there: e = the least exponent that takes the new
// tokens' largest finite value, and, where tokens of the same request lie in front of them in the block, at least the block's old one.
// If the old one was smaller, those tokens' codes are rounded to the new scale (exactly, for e4m3, down to its subnormals).  A warp owns
// a unit, (block of tokens, KV head, keys or values), from the largest value to the codes: no other warp touches that scale, so there is
// no atomic and no second launch.  The unit belongs to the first of its new rows: a row whose position is a block's first, or that is
// its request's first row.
//
// Bound by latency: description -> row -> old codes -> store, 2.4 us for 64 rows of 8 heads of 64 behind begun blocks; a prompt of 2,048 tokens
// 4.2 us (6.3 MB), 2,221 rows of 4 heads of 128 from float32 to integers 7.0 us (11.4 MB).  Up to CW_KEEP chunks of eight
// values a lane stay in registers between the two passes (16 tokens of 64 values: all of them); what is beyond is read again, from L1.
#define CW_WARPS 4
#define CW_KEEP 4

template <typename T, bool VEC>
__device__ __forceinline__ void cw_load8(const T* p, float (&x)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ng_ld(p + i);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ float cw_top(const float (&x)[8], float top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x[i]);
        top = a < __uint_as_float(0x7f800000u) ? fmaxf(top, a) : top;          // finite values only (NaN compares false)
    }
    return top;
}
template <int KIND>
__device__ __forceinline__ uint2 cw_codes(const float (&x)[8], float f) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = q8_from_float<KIND>(x[2 * i] * f, x[2 * i + 1] * f);
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// n chunks of eight codes, by a warp: to a scale that is 2^-by times theirs
template <int KIND>
__device__ __forceinline__ void cw_requantise(unsigned char* front, int n, int by) {
    const float g = q8_pow2(max(by, -126));                          // (below that every code becomes 0)
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        const uint2 w = *reinterpret_cast<const uint2*>(front + (size_t)i * 8);
        uint32_t h[4];
        q8_to_half<KIND>(w.x, h[0], h[1]);
        q8_to_half<KIND>(w.y, h[2], h[3]);
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(y[2 * j]), "=f"(y[2 * j + 1]) : "r"(h[j]));
        *reinterpret_cast<uint2*>(front + (size_t)i * 8) = cw_codes<KIND>(y, g);
    }
}

struct CwArgs {
    const void *k, *v;
    long long k_pitch, v_pitch;                     // elements between rows
    unsigned char *k_pages, *v_pages;
    float *k_scales, *v_scales;
    const int *table, *row_entry, *cu_q, *ctx_before;
    int* status;
    int table_stride, n_rows, n_entries, nKV, hd, ps_log2, bl_log2, num_pages, rows_per_block;
};

template <typename T, int KIND, bool VEC>
__global__ void __launch_bounds__(CW_WARPS * 32)
cache_write_q8_kernel(const CwArgs a) {
    ng_pdl_trigger();
    const int lane = threadIdx.x & 31, unit = blockIdx.y * CW_WARPS + (threadIdx.x >> 5);
    const int row0 = blockIdx.x * a.rows_per_block;
    const int block = 1 << a.bl_log2, mask = block - 1;
    // which of this block's rows (at most 32, one a lane) begin a unit
    int entry = -1, pos = 0, last = 0;
    bool leads = false;
    if (lane < a.rows_per_block && row0 + lane < a.n_rows) {
        entry = a.row_entry[row0 + lane];
        if (entry >= 0 && entry < a.n_entries) {
            const int first = a.cu_q[entry], ctx = a.ctx_before[entry];
            pos = ctx + row0 + lane - first;
            last = min(ctx + a.cu_q[entry + 1] - first, pos + a.n_rows - row0 - lane);      // rows that the buffers do not hold are not read
            leads = row0 + lane >= first && pos >= 0 && pos < last && (row0 + lane == first || (pos & mask) == 0);
        }
    }
    uint32_t todo = __ballot_sync(0xffffffffu, leads);
    ng_pdl_wait();
    if (unit >= 2 * a.nKV) return;
    const bool is_v = unit >= a.nKV;
    const int head = is_v ? unit - a.nKV : unit;
    const T* x = ng_after_wait(reinterpret_cast<const T*>(is_v ? a.v : a.k));
    const long long pitch = is_v ? a.v_pitch : a.k_pitch;
    unsigned char* pages = is_v ? a.v_pages : a.k_pages;
    float* scales = is_v ? a.v_scales : a.k_scales;
    const int per_row = a.hd >> 3;                  // chunks of eight values
    for (; todo; todo &= todo - 1) {
        const int at = __ffs(todo) - 1;
        const int e = __shfl_sync(0xffffffffu, entry, at), p0 = __shfl_sync(0xffffffffu, pos, at);
        const int end = min(__shfl_sync(0xffffffffu, last, at), (p0 | mask) + 1);        // behind the unit's last new token
        const int pi = p0 >> a.ps_log2;
        const int page = pi < a.table_stride ? a.table[(size_t)e * a.table_stride + pi] : -1;
        if (page < 0 || page >= a.num_pages) {
            if (lane == 0 && unit == 0) atomicOr(a.status, NG_STATUS_BAD_PAGE);
            continue;
        }
        const int slot = p0 & ((1 << a.ps_log2) - 1), lead = p0 & mask;        // tokens of the block that are already there
        const size_t slab = (size_t)page * a.nKV + head;
        unsigned char* dst = pages + ((slab << a.ps_log2) + slot) * a.hd;
        float* scale = scales + (slab << (a.ps_log2 - a.bl_log2)) + (slot >> a.bl_log2);
        const T* src = x + (long long)(row0 + at) * pitch + (long long)head * a.hd;
        const int n = (end - p0) * per_row;
        const int old = lead ? min(max(q8_exponent_of(*scale), NG_Q8_EXP_LOWEST), NG_Q8_EXP_HIGHEST) : NG_Q8_EXP_LOWEST;
        float keep[CW_KEEP][8], top = 0.f;
#pragma unroll
        for (int c = 0; c < CW_KEEP; ++c) {
            const int i = lane + 32 * c;
            if (i < n) cw_load8<T, VEC>(src + (i / per_row) * pitch + (i % per_row) * 8, keep[c]);
        }
#pragma unroll
        for (int c = 0; c < CW_KEEP; ++c)
            if (lane + 32 * c < n) top = cw_top(keep[c], top);
        for (int i = lane + 32 * CW_KEEP; i < n; i += 32) {
            float y[8];
            cw_load8<T, VEC>(src + (i / per_row) * pitch + (i % per_row) * 8, y);
            top = cw_top(y, top);
        }
        const int exp = max(q8_exponent<KIND>(ng_warp_max(top)), old);
        const float f = q8_pow2(-exp);
#pragma unroll
        for (int c = 0; c < CW_KEEP; ++c) {
            const int i = lane + 32 * c;
            if (i < n) *reinterpret_cast<uint2*>(dst + (size_t)i * 8) = cw_codes<KIND>(keep[c], f);      // a token's values follow the one before's
        }
        for (int i = lane + 32 * CW_KEEP; i < n; i += 32) {
            float y[8];
            cw_load8<T, VEC>(src + (i / per_row) * pitch + (i % per_row) * 8, y);
            *reinterpret_cast<uint2*>(dst + (size_t)i * 8) = cw_codes<KIND>(y, f);
        }
        if (lead && exp > old) cw_requantise<KIND>(dst - (size_t)lead * a.hd, lead * per_row, old - exp);
        __syncwarp();
        if (lane == 0 && (!lead || exp > old)) *scale = q8_pow2(exp);
    }
}

static int log2_of(int n) {
    int l = 0;
    while ((1 << l) < n) ++l;
    return l;
}
static bool power_of_two(int n) { return n > 0 && !(n & (n - 1)); }

// The arguments, packed (a call through ctypes pays for every argument: 26 of them took 5 us, a struct takes 1).
struct NgCacheWriteQ8 {
    const void *k, *v;
    void *k_pages, *v_pages;
    float *k_scales, *v_scales;
    const int *table, *row_entry, *cu_q, *ctx_before;
    int* status;
    long long k_pitch, v_pitch;                     // elements between rows
    int table_stride, n_rows, n_entries, n_kv, head_dim, page_size, block, num_pages, kind, in_bf16;
};
NG_EXPORT int ng_cache_write_q8(const NgCacheWriteQ8* c, cudaStream_t stream) {
    const int n_rows = c->n_rows, nKV = c->n_kv, kind = c->kind;
    if (n_rows <= 0 || c->n_entries <= 0) return NG_OK;
    if (nKV <= 0 || c->head_dim <= 0 || c->head_dim % 16 || !power_of_two(c->page_size) || !power_of_two(c->block) || c->block < 8 ||
        c->block > c->page_size || c->num_pages <= 0 || c->table_stride <= 0 || !c->status || (kind != NG_Q8_E4M3 && kind != NG_Q8_INT8) ||
        (((uintptr_t)c->k_pages | (uintptr_t)c->v_pages) & 7))
        return NG_BAD_SIZE;
    // Rows a block: single tokens one, for every row begins a unit and a block's units follow one another; prompts eight, for one row in `block`
    // does, and idle blocks cost too.  Heads of 64, 8 KV heads, one / eight, us: 64 single tokens 2.6 / 9.9, 512 5.8 / 10.6, 1,024 10.1 / 11.6;
    // a prompt of 256 tokens 3.6 / 3.3, 512 4.6 / 3.6, 2,048 10.8 / 4.6, 8,192 36.2 / 10.1
    const int rpb = n_rows < 8 * c->n_entries ? 1 : 8;
    const CwArgs a{c->k, c->v, c->k_pitch, c->v_pitch, (unsigned char*)c->k_pages, (unsigned char*)c->v_pages, c->k_scales, c->v_scales,
                   c->table, c->row_entry, c->cu_q, c->ctx_before, c->status, c->table_stride, n_rows, c->n_entries, nKV, c->head_dim,
                   log2_of(c->page_size), log2_of(c->block), c->num_pages, rpb};
    dim3 grid((n_rows + rpb - 1) / rpb, (2 * nKV + CW_WARPS - 1) / CW_WARPS);
    if (grid.y > 65535) return NG_BAD_SIZE;
    const int esz = c->in_bf16 ? 2 : 4;
    const bool vec = !(((uintptr_t)c->k | (uintptr_t)c->v) & 15) && c->k_pitch * esz % 16 == 0 && c->v_pitch * esz % 16 == 0;
#define CW_GO(T, KIND, VEC) NG_LAUNCH((cache_write_q8_kernel<T, KIND, VEC>), grid, CW_WARPS * 32, 0, stream, a)
#define CW_KINDS(T, VEC) do { if (kind == NG_Q8_E4M3) CW_GO(T, NG_Q8_E4M3, VEC); else CW_GO(T, NG_Q8_INT8, VEC); } while (0)
    if (c->in_bf16 && vec) CW_KINDS(__nv_bfloat16, true);
    else if (c->in_bf16) CW_KINDS(__nv_bfloat16, false);
    else if (vec) CW_KINDS(float, true);
    else CW_KINDS(float, false);
    return ng_launch_status();
}

// ===================================================================================== rotation and write of single tokens
// rope_cache.cu's preparation (a head's norm, the rotation, one rounding to bfloat16; the same arithmetic in the same order) and the write above in
// one launch, for steps whose entries bring one token each: a warp has a head, and so all that is new in its block.  6 layers of LFM2-1.2B a
// step: a launch of about 2.4 us less each.
struct NgRopeCacheQ8 {
    const void* qkv;                                // [rows, (heads + 2 KV heads) head_dim] in bfloat16, or n_part float32 partial sums of it
    void* q_out;
    const float *q_weight, *k_weight, *inv_freq;
    void *k_pages, *v_pages;
    float *k_scales, *v_scales;
    const int *table, *positions, *row_entry;
    int* status;
    long long part_stride;
    int n_part, half_pairing, table_stride, n_entries, n_rows, n_heads, n_kv, head_dim, page_size, block, num_pages, kind;
    float pos_scale, eps;
};
#define RQ_WARPS 4
template <typename TI, int KIND, int PAIRS>
__global__ void __launch_bounds__(RQ_WARPS * 32)
rope_cache_q8_kernel(const NgRopeCacheQ8 c, int ps_log2, int bl_log2) {
    ng_pdl_trigger();
    const int row = blockIdx.x, lane = threadIdx.x & 31, head = blockIdx.y * RQ_WARPS + (threadIdx.x >> 5);
    const int entry = c.row_entry[row], pos = c.positions[row], hd = c.head_dim, half = hd / 2;
    const bool is_q = head < c.n_heads, is_v = head >= c.n_heads + c.n_kv;
    const float* w = is_q ? c.q_weight : is_v ? nullptr : c.k_weight;
    const bool turn = c.inv_freq && !is_v;
    const float pf = (float)pos / c.pos_scale;
    int ia[PAIRS], ib[PAIRS];
    float sn[PAIRS], cs[PAIRS], wa[PAIRS], wb[PAIRS];
#pragma unroll
    for (int u = 0; u < PAIRS; ++u) {
        const int i = min(lane + 32 * u, half - 1);
        ia[u] = c.half_pairing ? i : 2 * i;
        ib[u] = c.half_pairing ? i + half : 2 * i + 1;
        sn[u] = 0.f;
        cs[u] = 1.f;
        if (turn && lane + 32 * u < half) sincosf(pf * c.inv_freq[i], &sn[u], &cs[u]);
        wa[u] = w ? w[ia[u]] : 1.f;
        wb[u] = w ? w[ib[u]] : 1.f;
    }
    ng_pdl_wait();
    if (head >= c.n_heads + 2 * c.n_kv) return;
    __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(c.q_out) + ((size_t)row * c.n_heads + head) * hd;
    if (entry < 0 || entry >= c.n_entries) {        // padding row: defined output, no cache write
        if (is_q)
            for (int j = lane; j < hd; j += 32) q[j] = __float2bfloat16(0.f);
        return;
    }
    const TI* in = ng_after_wait(reinterpret_cast<const TI*>(c.qkv)) + ((size_t)row * (c.n_heads + 2 * c.n_kv) + head) * hd;
    float x[PAIRS], y[PAIRS], ss = 0.f;
#pragma unroll
    for (int u = 0; u < PAIRS; ++u) {
        x[u] = ng_ld_sum<__nv_bfloat16>(in, ia[u], c.n_part, c.part_stride);
        y[u] = ng_ld_sum<__nv_bfloat16>(in, ib[u], c.n_part, c.part_stride);
        if (sizeof(TI) == 4) {                      // (a stack of one part is not rounded yet)
            x[u] = __bfloat162float(__float2bfloat16(x[u]));
            y[u] = __bfloat162float(__float2bfloat16(y[u]));
        }
        if (lane + 32 * u >= half) x[u] = y[u] = 0.f;
    }
    if (w) {
#pragma unroll
        for (int u = 0; u < PAIRS; ++u) ss += x[u] * x[u] + y[u] * y[u];
        const float r = rsqrtf(ng_warp_sum(ss) / (float)hd + c.eps);
#pragma unroll
        for (int u = 0; u < PAIRS; ++u) x[u] = x[u] * r * wa[u], y[u] = y[u] * r * wb[u];
    }
    float top = 0.f;
#pragma unroll
    for (int u = 0; u < PAIRS; ++u) {
        if (turn) {
            const float a = x[u] * cs[u] - y[u] * sn[u], b = x[u] * sn[u] + y[u] * cs[u];
            x[u] = a;
            y[u] = b;
        }
        const __nv_bfloat16 a = __float2bfloat16(x[u]), b = __float2bfloat16(y[u]);
        if (lane + 32 * u < half) {
            if (is_q) q[ia[u]] = a, q[ib[u]] = b;
            x[u] = __bfloat162float(a);
            y[u] = __bfloat162float(b);
            top = fabsf(x[u]) < INFINITY ? fmaxf(top, fabsf(x[u])) : top;
            top = fabsf(y[u]) < INFINITY ? fmaxf(top, fabsf(y[u])) : top;
        }
    }
    if (is_q) return;
    const int kv = is_v ? head - c.n_heads - c.n_kv : head - c.n_heads, pi = pos >> ps_log2;
    const int page = pos >= 0 && pi < c.table_stride ? c.table[(size_t)entry * c.table_stride + pi] : -1;
    if (page < 0 || page >= c.num_pages) {
        if (lane == 0 && head == c.n_heads) atomicOr(c.status, NG_STATUS_BAD_PAGE);
        return;
    }
    const int slot = pos & ((1 << ps_log2) - 1), lead = pos & ((1 << bl_log2) - 1);
    const size_t slab = (size_t)page * c.n_kv + kv;
    unsigned char* dst = reinterpret_cast<unsigned char*>(is_v ? c.v_pages : c.k_pages) + ((slab << ps_log2) + slot) * hd;
    float* scale = (is_v ? c.v_scales : c.k_scales) + (slab << (ps_log2 - bl_log2)) + (slot >> bl_log2);
    const int old = lead ? min(max(q8_exponent_of(*scale), NG_Q8_EXP_LOWEST), NG_Q8_EXP_HIGHEST) : NG_Q8_EXP_LOWEST;
    const int exp = max(q8_exponent<KIND>(ng_warp_max(top)), old);
    const float f = q8_pow2(-exp);
#pragma unroll
    for (int u = 0; u < PAIRS; ++u)
        if (lane + 32 * u < half) {
            const uint32_t h = q8_from_float<KIND>(x[u] * f, y[u] * f);
            dst[ia[u]] = (unsigned char)h;
            dst[ib[u]] = (unsigned char)(h >> 8);
        }
    if (lead && exp > old) cw_requantise<KIND>(dst - (size_t)lead * hd, lead * (hd >> 3), old - exp);
    __syncwarp();
    if (lane == 0 && (!lead || exp > old)) *scale = q8_pow2(exp);
}

NG_EXPORT int ng_rope_cache_q8(const NgRopeCacheQ8* call, cudaStream_t stream) {
    const NgRopeCacheQ8& c = *call;
    if (c.n_rows <= 0) return NG_OK;
    if (c.n_heads <= 0 || c.n_kv <= 0 || c.head_dim <= 0 || c.head_dim % 16 || c.head_dim > 256 || !power_of_two(c.page_size) ||
        !power_of_two(c.block) || c.block < 8 || c.block > c.page_size || c.num_pages <= 0 || c.table_stride <= 0 || !c.status || c.n_part < 0 ||
        c.pos_scale == 0.f || (c.kind != NG_Q8_E4M3 && c.kind != NG_Q8_INT8) || (((uintptr_t)c.k_pages | (uintptr_t)c.v_pages) & 7))
        return NG_BAD_SIZE;
    const dim3 grid(c.n_rows, (c.n_heads + 2 * c.n_kv + RQ_WARPS - 1) / RQ_WARPS);
    if (grid.y > 65535) return NG_BAD_SIZE;
#define RQ_GO(TI, KIND, PAIRS) NG_LAUNCH((rope_cache_q8_kernel<TI, KIND, PAIRS>), grid, RQ_WARPS * 32, 0, stream, c, log2_of(c.page_size), log2_of(c.block))
#define RQ_PAIRS(TI, KIND)                                                                                                             \
    do {                                                                                                                               \
        if (c.head_dim <= 64) RQ_GO(TI, KIND, 1);                                                                                      \
        else if (c.head_dim <= 128) RQ_GO(TI, KIND, 2);                                                                                \
        else RQ_GO(TI, KIND, 4);                                                                                                       \
    } while (0)
#define RQ_KINDS(TI) do { if (c.kind == NG_Q8_E4M3) RQ_PAIRS(TI, NG_Q8_E4M3); else RQ_PAIRS(TI, NG_Q8_INT8); } while (0)
    if (c.n_part > 0) RQ_KINDS(float);
    else RQ_KINDS(__nv_bfloat16);
    return ng_launch_status();
}

// ===================================================================================== copies of pages
// pool[layer, dst_i] = pool[layer, src_i] for every layer of up to CP_POOLS pools at once: keys, values and their scales in one launch.
// The page numbers travel as kernel parameters (no copy to the device in front of the kernel, nothing to keep alive behind it); they are
// host values, so the launcher checks them all before anything runs.
//
// Bound by bytes: every page is read and written once.  The copy of a layer is a row of 16-byte pieces (smaller where the pages'
// size or addresses ask for it), CP_UNROLL of them requested by a thread before the first is stored; which pair a piece belongs to is a
// multiplication by the inverse of the pieces a page has.  4,096 pages of 6 layers (8 heads of 64, e4m3 with scales, 808 MB moved): 134 us =
// 6.0 TB/s, 0.92 of a plain copy's rate; four pages 1.8 us.  Pieces a thread 2 / 4 / 8 / 16: 134 / 134 / 155 / 192 us (more of them leave fewer
// threads resident), with streaming loads and stores 136 / 150 / 156.
#define CP_POOLS 8
#define CP_UNROLL 2
#define CP_THREADS 256
enum { NG_BAD_PAGES = 6 };           // a page number is outside its pool, written twice, or both read and written

struct CpPool {
    unsigned char* base;
    long long layer_bytes;
    uint32_t pieces, piece_log2;     // of a page
    uint32_t inverse, shift;         // i / pieces = umulhi(i, inverse) >> shift, or i >> shift for a power of two (inverse 0)
    int first_tile, layers, tiles;   // tiles of a layer's copy; the pool's tiles follow those of the pool before
};
template <int N>
struct CpArgs {
    CpPool pool[CP_POOLS];
    int n_pools, n_pairs, n_tiles;
    int src[N], dst[N];
};

template <typename V, int N>
__device__ __forceinline__ void cp_tile(const CpArgs<N>& a, const CpPool& p, int tile) {
    const int layer = tile / p.tiles;
    const uint32_t first = (uint32_t)(tile - layer * p.tiles) * (CP_THREADS * CP_UNROLL) + threadIdx.x, total = p.pieces * a.n_pairs;
    unsigned char* base = p.base + layer * p.layer_bytes;
    V x[CP_UNROLL];
    V* to[CP_UNROLL];
#pragma unroll
    for (int u = 0; u < CP_UNROLL; ++u) {
        const uint32_t i = first + u * CP_THREADS;
        if (i >= total) continue;
        const uint32_t pair = p.inverse ? __umulhi(i, p.inverse) >> p.shift : i >> p.shift;
        const size_t piece = i - pair * p.pieces;
        x[u] = reinterpret_cast<const V*>(base)[(size_t)a.src[pair] * p.pieces + piece];
        to[u] = reinterpret_cast<V*>(base) + (size_t)a.dst[pair] * p.pieces + piece;
    }
#pragma unroll
    for (int u = 0; u < CP_UNROLL; ++u)
        if (first + u * CP_THREADS < total) *to[u] = x[u];
}

template <int N>
__global__ void __launch_bounds__(CP_THREADS)
copy_pages_kernel(const __grid_constant__ CpArgs<N> a) {
    ng_pdl_trigger();
    ng_pdl_wait();
    for (int tile = blockIdx.x; tile < a.n_tiles; tile += gridDim.x) {
        int k = 0;
        while (k + 1 < a.n_pools && tile >= a.pool[k + 1].first_tile) ++k;
        const CpPool& p = a.pool[k];
        switch (p.piece_log2) {
            case 4: cp_tile<uint4>(a, p, tile - p.first_tile); break;
            case 2: cp_tile<uint32_t>(a, p, tile - p.first_tile); break;
            default: cp_tile<unsigned char>(a, p, tile - p.first_tile);
        }
    }
}

template <int N>
static int cp_launch(CpPool* pools, int n_pools, const int* src, const int* dst, int n, cudaStream_t stream) {
    static thread_local CpArgs<N> a;
    long long tiles = 0;
    for (int k = 0; k < n_pools; ++k) {
        CpPool& p = pools[k];
        p.tiles = (int)(((long long)p.pieces * n + CP_THREADS * CP_UNROLL - 1) / (CP_THREADS * CP_UNROLL));
        p.first_tile = (int)tiles;
        tiles += (long long)p.tiles * p.layers;
        a.pool[k] = p;
    }
    if (tiles > 0x7fffffff) return NG_BAD_SIZE;
    a.n_pools = n_pools;
    a.n_pairs = n;
    a.n_tiles = (int)tiles;
    memcpy(a.src, src, n * sizeof(int));
    memcpy(a.dst, dst, n * sizeof(int));
    NG_LAUNCH((copy_pages_kernel<N>), dim3((unsigned)tiles), CP_THREADS, 0, stream, a);
    return NG_OK;
}

struct NgPool {
    void* base;
    long long page_bytes;
    int layers, pages;               // a layer's pages follow one another, and so do the layers
};
NG_EXPORT int ng_copy_pages(const NgPool* pool, int n_pools, const int* src, const int* dst, int n, cudaStream_t stream) {
    if (n < 0 || n_pools < 0 || n_pools > CP_POOLS) return NG_BAD_SIZE;
    if (n == 0 || n_pools == 0) return NG_OK;
    int fewest = 0x7fffffff;
    for (int k = 0; k < n_pools; ++k) {
        if (pool[k].layers < 0 || pool[k].pages < 0 || pool[k].page_bytes <= 0) return NG_BAD_SIZE;
        fewest = pool[k].pages < fewest ? pool[k].pages : fewest;
    }
    for (int i = 0; i < n; ++i)
        if (src[i] < 0 || src[i] >= fewest || dst[i] < 0 || dst[i] >= fewest) return NG_BAD_PAGES;
    if (n <= 16) {
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < n; ++j)
                if (dst[i] == src[j] || (i != j && dst[i] == dst[j])) return NG_BAD_PAGES;
    } else {
        unsigned char* seen = (unsigned char*)calloc(fewest, 1);
        if (!seen) return NG_BAD_SIZE;
        bool ok = true;
        for (int i = 0; i < n; ++i) ok &= !seen[dst[i]], seen[dst[i]] = 1;
        for (int i = 0; i < n; ++i) ok &= !seen[src[i]];
        free(seen);
        if (!ok) return NG_BAD_PAGES;
    }
    CpPool pools[CP_POOLS];
    for (int k = 0; k < n_pools; ++k) {
        CpPool& p = pools[k];
        p.base = (unsigned char*)pool[k].base;
        p.layers = pool[k].layers;
        p.layer_bytes = pool[k].page_bytes * pool[k].pages;
        const unsigned long long at = (uintptr_t)p.base | (unsigned long long)pool[k].page_bytes;        // layers are whole pages apart
        p.piece_log2 = at % 16 == 0 ? 4 : at % 4 == 0 ? 2 : 0;
        const long long pieces = pool[k].page_bytes >> p.piece_log2;
        if (pieces > (1 << 20)) return NG_BAD_SIZE;               // 1,024 pairs of them are counted in 31 bits
        p.pieces = (uint32_t)pieces;
        // i / pieces for i < 2^31, the round-up method: with 2^shift' >= pieces, m = ceil(2^(32 + s) / pieces), s = shift' - 1
        int s = 0;
        while ((1u << s) < p.pieces) ++s;
        if ((1u << s) == p.pieces) {
            p.inverse = 0;
            p.shift = s;
        } else {
            p.shift = s - 1;
            p.inverse = (uint32_t)(((1ull << (31 + s)) + p.pieces - 1) / p.pieces);
        }
    }
    for (int i = 0; i < n;) {
        const int left = n - i;
        int rc, took;
        if (left <= 32) took = left, rc = cp_launch<32>(pools, n_pools, src + i, dst + i, took, stream);
        else took = left < 1024 ? left : 1024, rc = cp_launch<1024>(pools, n_pools, src + i, dst + i, took, stream);
        if (rc != NG_OK) return rc;
        i += took;
    }
    return ng_launch_status();
}
