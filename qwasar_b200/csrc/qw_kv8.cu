// The 8-bit K/V cache: append, dequantising read, and attention over it (sm_100a).
//
// Format.  A key or value element is an e4m3 code times 2^e, with one e per 64 tokens of one head.  e is the
// smallest whole number for which the block's largest magnitude is at most 448 * 2^e, within [-60, 119]; its byte is
// e + 127.  Powers of two keep every step but the rounding to e4m3 exact: scaling by 2^-e, moving a block to a larger
// e when a bigger row arrives (a shift, exact until a code falls below the normal range), widening a code to fp16 or
// bf16 -- so attention can fold the exponents into the softmax instead of touching the elements.
#include "qw_kernels.h"
#include <algorithm>
#include <cuda_fp16.h>

namespace qw {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int BLK = QW_KV8_BLOCK;

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // e in [-126, 127]
__device__ __forceinline__ int clamp_exp(int byte) { return min(max(byte - 127, QW_KV8_E_MIN), QW_KV8_E_MAX); }
__device__ __forceinline__ int needed_exp(float amax) {
    // 448 = 1.75 * 2^8
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, QW_KV8_E_MIN), QW_KV8_E_MAX);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x4(const float *v) { return e4m3x2(v[0], v[1]) | (e4m3x2(v[2], v[3]) << 16); }
// two codes -> two fp16 values (exact)
__device__ __forceinline__ uint32_t f16x2_lo(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_hi(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ float2 h2f2(uint32_t h) {
    const __half2 v = *reinterpret_cast<const __half2 *>(&h);
    return __half22float2(v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Row of codes that holds (head, token), or -1 where no page is mapped.
__device__ __forceinline__ int64_t code_row(const Kv8Layer &L, int h, int t) {
    if (!L.table) return (int64_t)h * L.max_ctx + t;
    const int pg = __ldg(L.table + (size_t)h * L.pt_stride + t / QW_KV8_PAGE_TOKENS);
    return pg < 0 ? -1 : (int64_t)pg * QW_KV8_PAGE_TOKENS + (t & (QW_KV8_PAGE_TOKENS - 1));
}

// The same from a launch's fields (attention: one head of one sequence).
__device__ __forceinline__ int tile_row(const Kv8AttnParams &p, const int32_t *table, int h, int t) {
    if (!table) return h * p.max_ctx + t;
    const int pg = __ldg(table + (size_t)h * p.pt_stride + t / QW_KV8_PAGE_TOKENS);
    if (pg < 0) report(p.status, QW_ST_BAD_PAGE);
    return max(pg, 0) * QW_KV8_PAGE_TOKENS + (t & (QW_KV8_PAGE_TOKENS - 1));
}

// =======================================================================================
// append
// =======================================================================================
// One CTA per (64-token block, head, K or V, sequence): the block's new rows are read once into registers, their
// largest magnitude gives the exponent, and the codes leave as whole 256-byte rows.  A block that holds rows already
// keeps its exponent unless the new rows need a larger one; then its old codes are moved there first.  The exponent is
// known only when the last of the 64 rows is, so a CTA is one trip to memory, a reduction and the stores; what bounds it
// is that trip and, with few CTAs to an SM, how much of it is in flight: 4096 bf16 rows of
// 4 heads, K and V (16.8 MB in, 8.4 MB out), 4.7 us, one row 2.0 us (a trip for the old exponent and the rows together, and
// where the exponent grew one more for the old codes).
constexpr int WR_THREADS = 512, WR_WARPS = WR_THREADS / 32, WR_ROWS = BLK / WR_WARPS;

// Largest of `v` over the block; the same for every thread.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *red) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();                                         // (of the last use of `red`)
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < WR_WARPS; i++) v = max(v, red[i]);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(WR_THREADS) kv8_write_kernel(const __grid_constant__ Kv8WriteParams p) {
    __shared__ uint32_t red[WR_WARPS];
    pdl_wait();
    pdl_launch_next();
    const int h = blockIdx.y >> 1, which = blockIdx.y & 1;
    const Kv8WriteSeq &sq = p.seq[blockIdx.z];
    const int blk = sq.base_pos / BLK + (int)blockIdx.x, t0 = blk * BLK;
    const int first = max(t0, sq.base_pos), last = min(t0 + BLK, sq.base_pos + p.rows);   // new rows of this block
    if (first >= last) return;
    const Kv8Layer &L = which ? sq.vc : sq.kc;
    const T *src = reinterpret_cast<const T *>(which ? sq.v : sq.k) + (size_t)h * 256;
    const int col = (threadIdx.x & 31) * 8, r0 = first + (threadIdx.x >> 5);

    // all of the thread's rows are asked for before the first is looked at: one trip to memory
    constexpr int RW = sizeof(T) == 2 ? 4 : 8;               // words of eight elements
    uint32_t raw[WR_ROWS][RW];
#pragma unroll
    for (int i = 0; i < WR_ROWS; i++) {
        const int t = r0 + WR_WARPS * i;
        const uint4 *g = reinterpret_cast<const uint4 *>(src + (size_t)(t - sq.base_pos) * p.row_stride + col);
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (t < last) { a = g[0]; if (RW == 8) b = g[1]; }
        raw[i][0] = a.x; raw[i][1] = a.y; raw[i][2] = a.z; raw[i][3] = a.w;
        if constexpr (RW == 8) { raw[i][4] = b.x; raw[i][5] = b.y; raw[i][6] = b.z; raw[i][7] = b.w; }
    }
    const int64_t row0 = code_row(L, h, t0);                 // a block never crosses a page
    uint8_t *ep = L.exps + (size_t)h * L.exp_stride + blk;
    const int was = first > t0 ? clamp_exp(*ep) : QW_KV8_E_MIN;
    if (row0 < 0) { if (threadIdx.x == 0) report(p.status, QW_ST_BAD_PAGE); return; }
    uint8_t *dst = L.base + row0 * 256;
    auto element = [&](int i, int e) {
        if constexpr (RW == 8) return __uint_as_float(raw[i][e]);
        else return __uint_as_float((e & 1) ? raw[i][e >> 1] & 0xffff0000u : raw[i][e >> 1] << 16);
    };
    // magnitudes order like their bits: the largest as a whole number, in the upper half for bf16
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < WR_ROWS; i++)
#pragma unroll
        for (int k = 0; k < RW; k++) big = RW == 8 ? max(big, raw[i][k] & 0x7fffffffu) : __vmaxu2(big, raw[i][k] & 0x7fff7fffu);
    if constexpr (RW == 4) big = max(big & 0xffff0000u, big << 16);
    // (block_max lies between reading the stored exponent and replacing it)
    big = block_max(big, red);
    const bool odd = big >= 0x7f800000u;                     // a NaN or an infinity among them: the largest of the others
    if (odd) {
        if (threadIdx.x == 0) report(p.status, QW_ST_KV8_NONFINITE);
        big = 0;
#pragma unroll
        for (int i = 0; i < WR_ROWS; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint32_t u = __float_as_uint(element(i, k)) & 0x7fffffffu;
                big = max(big, u < 0x7f800000u ? u : 0u);
            }
        big = block_max(big, red);
    }
    const int e = max(was, needed_exp(__uint_as_float(big)));
    if (first > t0 && e > was) {
        // rows [t0, first): 16 codes to a thread
        const float f = pow2f(max(was - e, -126));
        for (int i = threadIdx.x; i < (first - t0) * 16; i += WR_THREADS) {
            uint4 *at = reinterpret_cast<uint4 *>(dst + (size_t)i * 16);
            uint4 q = *at;
            uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float2 a = h2f2(f16x2_lo(w[k])), b = h2f2(f16x2_hi(w[k]));
                w[k] = e4m3x2(a.x * f, a.y * f) | (e4m3x2(b.x * f, b.y * f) << 16);
            }
            *at = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    const float inv = pow2f(-e);
#pragma unroll
    for (int i = 0; i < WR_ROWS; i++) {
        const int t = r0 + WR_WARPS * i;
        if (t >= last) break;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = element(i, k) * inv;
        if (odd) {                                           // NaN: stored as zero; infinite: the largest code
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = v[k] == v[k] ? v[k] : 0.0f;
        }
        *reinterpret_cast<uint2 *>(dst + (size_t)(t - t0) * 256 + col) = make_uint2(e4m3x4(v), e4m3x4(v + 4));
    }
    if (threadIdx.x == 0) *ep = (uint8_t)(e + 127);
}

// =======================================================================================
// dequantising read
// =======================================================================================
// A warp takes whole rows (32 lanes x 8 codes), RD_ROWS of them in flight; 1 byte in, 2 or 4 out per element, so the
// stores are what bounds it: 131 072 rows to bf16 17.0 us (5.9 TB/s) with four rows, 17.4 with two; 2002 rows to f32, where
// a call is one trip to memory long, 1.9 us with two, 2.7 with four, 4.4 with eight.
constexpr int RD_THREADS = 256;

template <typename T, int RD_ROWS>
__global__ void __launch_bounds__(RD_THREADS) kv8_read_kernel(T *__restrict__ dst, const Kv8Layer L, int pos0, int n) {
    pdl_wait();
    pdl_launch_next();
    const int h = blockIdx.y, lane = threadIdx.x & 31;
    const int r0 = ((int)blockIdx.x * (RD_THREADS / 32) + (int)(threadIdx.x >> 5)) * RD_ROWS;
    uint2 q[RD_ROWS];
    float s[RD_ROWS];
#pragma unroll
    for (int i = 0; i < RD_ROWS; i++) {
        q[i] = make_uint2(0, 0); s[i] = 0.0f;
        if (r0 + i < n) {
            const int t = pos0 + r0 + i;
            const int64_t row = code_row(L, h, t);
            if (row >= 0) {
                q[i] = *reinterpret_cast<const uint2 *>(L.base + row * 256 + lane * 8);
                s[i] = pow2f(clamp_exp(L.exps[(size_t)h * L.exp_stride + t / BLK]));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RD_ROWS; i++) {
        if (r0 + i >= n) break;
        float2 v[4] = {h2f2(f16x2_lo(q[i].x)), h2f2(f16x2_hi(q[i].x)), h2f2(f16x2_lo(q[i].y)), h2f2(f16x2_hi(q[i].y))};
#pragma unroll
        for (int k = 0; k < 4; k++) { v[k].x *= s[i]; v[k].y *= s[i]; }
        T *o = dst + ((size_t)h * n + r0 + i) * 256 + lane * 8;
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint4 *>(o) = make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y), pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
        } else {
            *reinterpret_cast<float4 *>(o) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
            *reinterpret_cast<float4 *>(o + 4) = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
        }
    }
}

// =======================================================================================
// attention, few query rows: split over the keys
// =======================================================================================
// All (sequence, kv head) groups of a launch lie end to end as one line of 32-key tiles, cut into shares of equal
// cost, one per CTA (one CTA per SM); a share that crosses a group's end is taken as two segments.  The tiles of a
// segment are dealt to the CTA's warps, each of which keeps its own running maximum, sum and output; the warps are
// added up through shared memory at the segment's end, the CTAs of a cut group by a second kernel.
//
// The products are turned over: S^T = K Q^T and O^T = V^T P^T, so that the cache is the 16-row operand of the tensor
// op and the query rows are its eight columns.  With Q as the 16-row operand half of every op of a decode step would
// multiply padding, and the running output would take twice the registers.  (tcgen05 has no use here: its smallest tile is
// 64 rows, 6 of which a decode step of 24 heads over 4 would fill.)  Query row i = r * gqa + g of the group:
// all query heads of the kv head, all rows of the call.
//
// Types.  fp16 tensor ops, because an e4m3 code is an fp16 number exactly.  bf16 rows are exact in fp16 after scaling
// by a power of two.  f32 rows are cut into a high and a low fp16 part (22 bits) that go through the same accumulators
// one after the other; so are the softmax weights.  (Weights run up to 2^14, not 1, so that the small ones of a long
// context stay above fp16's smallest number: 2^-38 of the largest.)
//
// Exponents.  A tile of 32 keys has one exponent for K and one for V.  With t = scale * log2(e) * 2^ek * (q . ck) + ev
// and m the running maximum of t, w = 2^(t - m) weighs the V CODES: o = sum w cv, and the denominator is
// l = sum w 2^-ev.  Both see each element once, as it lies in the cache.
//
// Fragments.  A lane reads 16 bytes of one key (16 dims: four k-steps) or 16 dims of one key of V; keys are dealt to
// lanes so that the eight lanes of a shared-memory phase meet eight different bank groups of the SWIZZLE_128B boxes.
// The two keys of a V register are interleaved byte by byte before they are widened.  The weights come out with a key
// per lane group and are wanted with a query row there: movmatrix turns an 8 x 8 block.
constexpr int TILE = 32;
constexpr int ENTRY = TILE * 256;                    // K or V codes of a tile
constexpr int BOX = TILE * 128;
constexpr float W_SHIFT = 14.0f;
constexpr int SEG_COST = 8;                          // what a segment costs beside its tiles, in tiles (see kv8_attn_plan)

struct Where { int s, h, t; };                       // sequence, kv head, tile of the group

// The CTA whose share holds tile T: the last one that starts at or before it.
__host__ __device__ __forceinline__ int share_of(const Kv8AttnParams &p, int T) {
    int c = 0, e = p.n_cta - 1;
    while (c < e) {
        const int m = (c + e + 1) >> 1;
        if (p.share[m] <= T) c = m; else e = m - 1;
    }
    return c;
}
__device__ __forceinline__ Where locate(const Kv8AttnParams &p, int T) {
    int s = 0, e = p.n_seq - 1;
    while (s < e) {
        const int m = (s + e + 1) >> 1;
        if (p.seq[m].cum_tiles <= T) s = m; else e = m - 1;
    }
    const int rel = T - p.seq[s].cum_tiles, n = p.seq[s].n_tiles;
    Where w;
    w.s = s; w.h = rel / n; w.t = rel - w.h * n;
    return w;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float load1(const void *g, size_t i, int io) {
    return io == DT_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(g)[i]) : reinterpret_cast<const float *>(g)[i];
}
// Four finished dims of one row: divided by the denominator already; gated and stored.
__device__ __forceinline__ void store_out(const Kv8AttnParams &p, const Kv8AttnSeq &sq, size_t rh, int d4, float4 o) {
    if (sq.gate) {
        const size_t gi = rh * p.gate_stride + d4;
        o.x /= 1.0f + __expf(-load1(sq.gate, gi, p.io)); o.y /= 1.0f + __expf(-load1(sq.gate, gi + 1, p.io));
        o.z /= 1.0f + __expf(-load1(sq.gate, gi + 2, p.io)); o.w /= 1.0f + __expf(-load1(sq.gate, gi + 3, p.io));
    }
    if (p.io == DT_BF16)
        *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(sq.out) + rh * 256 + d4) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
    else
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(sq.out) + rh * 256 + d4) = o;
}

// =======================================================================================
// attention, up to eight query rows (a decode step)
// =======================================================================================
// A warp takes whole tiles: K in one 8 KB slot of its own, V in another, each refilled as soon as it is read, so that
// the other's load runs under its arithmetic.  The running output is 64 registers a thread; twelve warps fit an SM.
// Memory bounds the long calls: eight sequences of 32 K keys, 24 heads over 4 (537 MB) 88 us, 6.1 TB/s, of which a plain read
// of the same bytes takes 79; one sequence of 262 K keys 48.4 us of 43.5.  The short ones are a chain of trips: 4 K keys
// 8.3 us with the merge, of which the 8.4 MB take 1.3.
constexpr int D_WARPS = 12, D_THREADS = D_WARPS * 32, D_NS = 2;
constexpr int D_OFF_Q = D_WARPS * D_NS * ENTRY;
constexpr int D_OFF_M = D_OFF_Q + 8192;                   // [warp][8]
constexpr int D_OFF_L = D_OFF_M + D_WARPS * 32;
constexpr int D_OFF_SC = D_OFF_L + D_WARPS * 32;          // [8]
constexpr int D_OFF_T = D_OFF_SC + 32;                    // [2][8] maximum and sum of all warps
constexpr int D_OFF_BAR = D_OFF_T + 64;                   // full[warps * slots], abort
constexpr int D_SMEM = D_OFF_BAR + D_WARPS * D_NS * 8 + 16;
static_assert(D_SMEM <= 232448, "exceeds the 227 KB a CTA may use");

__device__ __forceinline__ uint32_t movm(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void lds128(uint32_t (&v)[4], uint32_t addr) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr));
}

__device__ __forceinline__ void l2_box(const CUtensorMap *map, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

// Query row `row` of a group, 8 dims per lane, as it lies in memory.  A segment asks for its query rows BEFORE it asks for
// keys and values: behind 200 KB of those per SM the rows came back 5 us later.
template <bool F32>
struct RowRaw { uint4 a, b; };
template <bool F32>
__device__ __forceinline__ RowRaw<F32> fetch_q(const Kv8AttnParams &p, const Kv8AttnSeq &sq, int head0, int valid, int row, int lane) {
    RowRaw<F32> x;
    x.a = x.b = make_uint4(0, 0, 0, 0);
    if (row < valid) {
        const int r = row / p.gqa, hh = row - r * p.gqa;
        const size_t at = ((size_t)r * p.q_heads + head0 + hh) * 256 + lane * 8;
        const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(sq.q) + at * (F32 ? 4 : 2));
        x.a = src[0];
        if (F32) x.b = src[1];
    }
    return x;
}
// Brings the query rows of the group a CTA turns to next (and a whole group's gate rows) into L2.
__device__ __forceinline__ void prefetch_rows(const void *base, int io, size_t row0_el, size_t row_stride_el, int rows_of_call, int gqa, int q_heads, int i, int lane) {
    if (i >= rows_of_call * gqa) return;
    const int r = i / gqa, hh = i - r * gqa;
    const size_t el = io == DT_F32 ? 4 : 2;
    const uint8_t *at = reinterpret_cast<const uint8_t *>(base) + (row0_el + ((size_t)r * q_heads + hh) * row_stride_el) * el + lane * 8 * el;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
}
// In front of the wait for the kernel before this one: what the CTA asks for first is brought into L2, under that kernel's
// tail.  Nothing is read here but page tables, which no kernel writes; a line that the kernel before still writes is in L2
// either way.  (Eight sequences of 32 K keys 88.3 us against 91.2, 262 K keys 48.4 against 49.7, 4 K 8.3 against 8.7; four tokens
// behind 32 K 26.0 against 26.7, in f32 31.5 against 33.1.)  A decode warp takes tiles whole
// (ROWS_K 32), a verify warp 16 keys of K and 128 dims of V.
template <int ROWS_K>
__device__ __forceinline__ void warm_tile(const Kv8AttnParams &p, const Kv8AttnSeq &sq, int h, int tile, int k_rows0, int v_col0, int lane) {
    const int key = tile * 32;
    auto row_of = [&](const int32_t *table) {
        if (!table) return h * p.max_ctx + key;
        const int pg = __ldg(table + (size_t)h * p.pt_stride + key / QW_KV8_PAGE_TOKENS);
        return pg < 0 ? -1 : pg * QW_KV8_PAGE_TOKENS + (key & (QW_KV8_PAGE_TOKENS - 1));
    };
    const int rk = row_of(sq.ktab), rv = row_of(sq.vtab);
    const size_t e = (size_t)h * p.exp_stride + key / BLK;
    if (lane == 0 && rk >= 0) {
        l2_box(&p.maps[sq.kmap], 0, rk + k_rows0); l2_box(&p.maps[sq.kmap], 128, rk + k_rows0);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(sq.kexp + e));
    }
    if (lane == 0 && rv >= 0) {
        if (ROWS_K == 32) { l2_box(&p.maps[sq.vmap], 0, rv); l2_box(&p.maps[sq.vmap], 128, rv); }
        else { l2_box(&p.maps[sq.vmap], v_col0, rv); l2_box(&p.maps[sq.vmap], v_col0, rv + 16); }
        asm volatile("prefetch.global.L2 [%0];" ::"l"(sq.vexp + e));
    }
}
// One warp stages a row: scaled below 2^14 and put where the B fragments are read: step 4 q + i takes dims
// 64 q + 16 t + 4 i + {0, 1 | 2, 3} of row g in lane (g, t).  `frags`: per tile of eight rows 8 pairs of steps x 32 lanes x
// 16 bytes (f32: 16 steps, high and low parts).  sc: scale * log2(e) * the row's 2^qe.
template <bool F32>
__device__ __forceinline__ void stage_q(const Kv8AttnParams &p, const RowRaw<F32> &raw, int row, int lane, uint8_t *frags, float *sc) {
    float x[8];
    if constexpr (F32) {
        x[0] = __uint_as_float(raw.a.x); x[1] = __uint_as_float(raw.a.y); x[2] = __uint_as_float(raw.a.z); x[3] = __uint_as_float(raw.a.w);
        x[4] = __uint_as_float(raw.b.x); x[5] = __uint_as_float(raw.b.y); x[6] = __uint_as_float(raw.b.z); x[7] = __uint_as_float(raw.b.w);
    } else {
        const uint32_t u[4] = {raw.a.x, raw.a.y, raw.a.z, raw.a.w};
#pragma unroll
        for (int k = 0; k < 4; k++) { x[2 * k] = __uint_as_float(u[k] << 16); x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u); }
    }
    float mx = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) mx = fmaxf(mx, fabsf(x[k]));
    mx = warp_max(mx);
    const int qe = min(max((int)(__float_as_uint(mx) >> 23) - 127 - 13, -100), 100);
    const float f = pow2f(-qe);
    if (lane == 0) *sc = p.scale * LOG2E * pow2f(qe);
    uint32_t hp[4];
#pragma unroll
    for (int k = 0; k < 4; k++) { x[2 * k] *= f; x[2 * k + 1] *= f; hp[k] = pack_f16(x[2 * k], x[2 * k + 1]); }
    const int q = lane >> 3, at = (row & 7) * 4 + ((lane >> 1) & 3);
    uint4 *fr = reinterpret_cast<uint4 *>(frags) + (row >> 3) * (F32 ? 512 : 256);
    if constexpr (F32) {
        uint32_t lp[4];
#pragma unroll
        for (int k = 0; k < 4; k++) { const float2 h = h2f2(hp[k]); lp[k] = pack_f16(x[2 * k] - h.x, x[2 * k + 1] - h.y); }
        fr[(q * 4 + (lane & 1) * 2) * 32 + at] = make_uint4(hp[0], hp[1], lp[0], lp[1]);
        fr[(q * 4 + (lane & 1) * 2 + 1) * 32 + at] = make_uint4(hp[2], hp[3], lp[2], lp[3]);
    } else {
        fr[(q * 2 + (lane & 1)) * 32 + at] = make_uint4(hp[0], hp[1], hp[2], hp[3]);
    }
}

// What this CTA reads later on and nothing hides: the gate rows of a group it finishes by itself, the query rows of the
// group after it.  Row i of either.
__device__ __forceinline__ void next_rows(const Kv8AttnParams &p, Where w, const Kv8AttnSeq &sq, int seg_t0, int seg_n, int T, int hi, int i, int lane) {
    if (sq.gate && seg_t0 == 0 && seg_n == sq.n_tiles)
        prefetch_rows(sq.gate, p.io, (size_t)w.h * p.gqa * p.gate_stride, p.gate_stride, sq.rows, p.gqa, p.q_heads, i, lane);
    if (T + seg_n < hi) {
        if (++w.h == p.kv_heads) { w.h = 0; w.s++; }
        const Kv8AttnSeq &nx = p.seq[w.s];
        prefetch_rows(nx.q, p.io, (size_t)w.h * p.gqa * 256, 256, nx.rows, p.gqa, p.q_heads, i, lane);
    }
}

template <bool F32>
__global__ void __launch_bounds__(D_THREADS, 1) kv8_decode_kernel(const __grid_constant__ Kv8AttnParams p) {
    constexpr int KG = D_WARPS, NS = D_NS;
    extern __shared__ __align__(1024) uint8_t smem[];
    float *sm_m = reinterpret_cast<float *>(smem + D_OFF_M);
    float *sm_l = reinterpret_cast<float *>(smem + D_OFF_L);
    float *sm_sc = reinterpret_cast<float *>(smem + D_OFF_SC);
    float *sm_t = reinterpret_cast<float *>(smem + D_OFF_T);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + D_OFF_BAR);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(full + KG * NS);

    if (smem_u32(smem) & 1023u) {                    // swizzled boxes need 1024-byte alignment
        if (threadIdx.x == 0) report(p.status, QW_ST_BAD_SMEM);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) {
        for (int i = 0; i < KG * NS; i++) mbar_init(&full[i], 1);
        *abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&p.maps[0]);
        tma_prefetch_desc(&p.maps[1]);
    }
    const int lo = p.share[blockIdx.x], hi = p.share[blockIdx.x + 1];
    Where w = locate(p, lo);
    {
        const Kv8AttnSeq &sq = p.seq[w.s];
        if (warp < 8) prefetch_rows(sq.q, p.io, (size_t)w.h * p.gqa * 256, 256, sq.rows, p.gqa, p.q_heads, warp, lane);
        if (warp < min(sq.n_tiles - w.t, hi - lo)) warm_tile<32>(p, sq, w.h, w.t + warp, 0, 0, lane);
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_next();

    uint8_t *ring = smem + warp * NS * ENTRY;
    full += warp * NS;
    uint32_t phase = 0;                              // of both slots: K in slot 0, V in slot 1

    auto load = [&](const Kv8AttnSeq &sq, int row, int is_v) {       // lane 0
        mbar_expect_tx(&full[is_v], ENTRY);
        const CUtensorMap *map = &p.maps[is_v ? sq.vmap : sq.kmap];
        tma_load_2d(ring + is_v * ENTRY, map, 0, row, &full[is_v]);
        tma_load_2d(ring + is_v * ENTRY + BOX, map, 128, row, &full[is_v]);
    };
    for (int T = lo; T < hi;) {
        const Kv8AttnSeq &sq = p.seq[w.s];
        const int seg_t0 = w.t, seg_n = min(sq.n_tiles - w.t, hi - T);
        const int valid = sq.rows * p.gqa, head0 = w.h * p.gqa;
        const int n_keys = sq.base_pos + sq.rows;
        const int nt = warp < seg_n ? (seg_n - warp + KG - 1) / KG : 0;      // this warp's tiles

        int win_k = 0, win_v = 0, win_e = 0;         // code rows and exponents of 32 tiles, one per lane
        auto window = [&](int i0) {
            const int i = i0 + lane;
            if (i < nt) {
                const int key = (seg_t0 + warp + i * KG) * TILE;
                win_k = tile_row(p, sq.ktab, w.h, key); win_v = tile_row(p, sq.vtab, w.h, key);
                const int ek = clamp_exp(sq.kexp[(size_t)w.h * p.exp_stride + key / BLK]);
                const int ev = clamp_exp(sq.vexp[(size_t)w.h * p.exp_stride + key / BLK]);
                win_e = (ek & 0xffff) | (ev << 16);
            }
        };
        RowRaw<F32> raw;
        if (warp < 8) raw = fetch_q<F32>(p, sq, head0, valid, warp, lane);
        if (nt > 0) {
            window(0);
            if (lane == 0) { load(sq, win_k, 0); load(sq, win_v, 1); }
        }
        if (warp < 8) next_rows(p, w, sq, seg_t0, seg_n, T, hi, warp, lane);

        if (warp < 8) stage_q<F32>(p, raw, warp, lane, smem + D_OFF_Q, sm_sc + warp);
        __syncthreads();

        float o[16][4];
#pragma unroll
        for (int n = 0; n < 16; n++) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f; }
        // this thread's columns: query rows 2 t and 2 t + 1
        const int row0 = 2 * t, row1 = row0 + 1;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        const int lim0 = row0 < valid ? sq.base_pos + row0 / p.gqa : n_keys - 1;
        const int lim1 = row1 < valid ? sq.base_pos + row1 / p.gqa : n_keys - 1;
        const float sc0 = sm_sc[row0], sc1 = sm_sc[row1];
        const uint32_t q_base = smem_u32(smem + D_OFF_Q) + lane * 16;
        const uint32_t tok = (uint32_t)(g ^ ((g & 1) << 2));         // this lane group's key of a block of eight
        const uint32_t k_base = smem_u32(ring) + tok * 128, v_base = smem_u32(ring + ENTRY);

#pragma unroll 1
        for (int i = 0; i < nt; i++, phase ^= 1) {
            const int key0 = (seg_t0 + warp + i * KG) * TILE;
            const int ex = __shfl_sync(0xffffffffu, win_e, i & 31);
            const int ek = (int)(int16_t)(ex & 0xffff), ev = ex >> 16;
            if (i + 1 < nt && ((i + 1) & 31) == 0) window(i + 1);
            const int nk = __shfl_sync(0xffffffffu, win_k, (i + 1) & 31), nv = __shfl_sync(0xffffffffu, win_v, (i + 1) & 31);

            // ---- S^T = K Q^T ----
            // (f32: the tensor op's running sum loses a little at every step, so the high parts of even and odd steps and
            // the low parts have sums of their own)
            float s[2][4], s1[2][4], sl[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[n][c] = s1[n][c] = sl[n][c] = 0.0f;
            mbar_wait(&full[0], phase, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint32_t kw[4][4];                     // keys tok, tok + 8, tok + 16, tok + 24
#pragma unroll
                for (int n = 0; n < 4; n++) lds128(kw[n], k_base + (q >> 1) * BOX + n * 1024 + ((((uint32_t)(4 * (q & 1) + t)) ^ tok) << 4));
#pragma unroll
                for (int kk = 0; kk < 2; kk++) {
                    uint32_t qf[2][4];
                    if constexpr (F32) { lds128(qf[0], q_base + (q * 4 + kk * 2) * 512); lds128(qf[1], q_base + (q * 4 + kk * 2 + 1) * 512); }
                    else lds128(qf[0], q_base + (q * 2 + kk) * 512);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int k = kk * 2 + h;
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            const uint32_t a0 = f16x2_lo(kw[2 * n][k]), a1 = f16x2_lo(kw[2 * n + 1][k]), a2 = f16x2_hi(kw[2 * n][k]), a3 = f16x2_hi(kw[2 * n + 1][k]);
                            if constexpr (F32) {
                                mma_f16(h ? s1[n] : s[n], a0, a1, a2, a3, qf[h][0], qf[h][1]);
                                mma_f16(sl[n], a0, a1, a2, a3, qf[h][2], qf[h][3]);
                            } else {
                                mma_f16(s[n], a0, a1, a2, a3, qf[0][2 * h], qf[0][2 * h + 1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && i + 1 < nt) load(sq, nk, 0);

            // ---- online softmax ----
            if constexpr (F32) {
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) s[n][c] += s1[n][c] + sl[n][c];
            }
            const float k0 = sc0 * pow2f(ek), k1 = sc1 * pow2f(ek), fv = (float)ev;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[n][c] = fmaf(s[n][c], (c & 1) ? k1 : k0, fv);
            if (key0 + TILE > sq.base_pos + 1) {
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (key0 + n * 16 + (c >> 1) * 8 + (int)tok > ((c & 1) ? lim1 : lim0)) s[n][c] = -INFINITY;
            }
            float x0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
            float x1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
            }
            if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
                const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
                const float f0 = m0 == n0 ? 1.0f : ex2(m0 - n0), f1 = m1 == n1 ? 1.0f : ex2(m1 - n1);
                l0 *= f0; l1 *= f1;
#pragma unroll
                for (int n = 0; n < 16; n++) { o[n][0] *= f0; o[n][1] *= f1; o[n][2] *= f0; o[n][3] *= f1; }
                m0 = n0; m1 = n1;
            }
            const float b0 = (m0 == -INFINITY ? 0.0f : m0) - W_SHIFT, b1 = (m1 == -INFINITY ? 0.0f : m1) - W_SHIFT;
            uint32_t pb[2][2], pl[2][2];               // B fragments of the weights (f32: high and low parts)
            float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float w0 = ex2(s[n][2 * c] - b0), w1 = ex2(s[n][2 * c + 1] - b1);
                    a0 += w0; a1 += w1;
                    const uint32_t hi = pack_f16(w0, w1);
                    pb[n][c] = movm(hi);
                    if constexpr (F32) {
                        const float2 h = h2f2(hi);
                        pl[n][c] = movm(pack_f16(w0 - h.x, w1 - h.y));
                    }
                }
            const float iv = pow2f(-ev);
            l0 = fmaf(a0, iv, l0); l1 = fmaf(a1, iv, l1);

            // ---- O^T += V^T P^T: row g of tile 8 x + j is dim 128 x + 16 g + 2 j, row g + 8 the dim after it; the two
            // keys of a register are interleaved byte by byte before they are widened ----
            mbar_wait(&full[1], phase, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
            if (key0 + TILE > n_keys) {                // rows past the last key may hold anything
                for (int off = (n_keys - key0) * 128 + lane * 16; off < TILE * 128; off += 512) {
                    *reinterpret_cast<uint4 *>(ring + ENTRY + off) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(ring + ENTRY + BOX + off) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
            }
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const uint32_t ta = 16 * n + 2 * t, tb = 16 * n + ((2 * t + 1) ^ 4);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    uint32_t v[4][4];                  // keys ta, tb, ta + 8, tb + 8
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const uint32_t tk = ((c & 1) ? tb : ta) + (c >> 1) * 8;
                        lds128(v[c], v_base + x * BOX + tk * 128 + (((uint32_t)g ^ (tk & 7)) << 4));
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t p0 = __byte_perm(v[0][k], v[1][k], 0x5140), p1 = __byte_perm(v[0][k], v[1][k], 0x7362);
                        const uint32_t r0 = __byte_perm(v[2][k], v[3][k], 0x5140), r1 = __byte_perm(v[2][k], v[3][k], 0x7362);
                        const uint32_t c0 = f16x2_lo(p0), c1 = f16x2_hi(p0), c2 = f16x2_lo(r0), c3 = f16x2_hi(r0);
                        const uint32_t d0 = f16x2_lo(p1), d1 = f16x2_hi(p1), d2 = f16x2_lo(r1), d3 = f16x2_hi(r1);
                        mma_f16(o[x * 8 + 2 * k], c0, c1, c2, c3, pb[n][0], pb[n][1]);
                        mma_f16(o[x * 8 + 2 * k + 1], d0, d1, d2, d3, pb[n][0], pb[n][1]);
                        if constexpr (F32) {
                            mma_f16(o[x * 8 + 2 * k], c0, c1, c2, c3, pl[n][0], pl[n][1]);
                            mma_f16(o[x * 8 + 2 * k + 1], d0, d1, d2, d3, pl[n][0], pl[n][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && i + 1 < nt) load(sq, nv, 1);
        }

        // ---- segment end: every warp puts its sums into its first slot, and all threads add them up ----
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        if (g == 0) { sm_m[warp * 8 + row0] = m0; sm_m[warp * 8 + row1] = m1; sm_l[warp * 8 + row0] = l0; sm_l[warp * 8 + row1] = l1; }
        if (nt > 0) {
            // piece c (four dims) of a row sits at c ^ ((row >> 1) & 3), which spreads a phase's eight lanes over the banks
            float *own = reinterpret_cast<float *>(ring);
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int n = x * 8 + 2 * e;
                    const uint32_t piece = (uint32_t)(x * 32 + g * 4 + e) ^ (uint32_t)t;
                    *reinterpret_cast<float4 *>(own + row0 * 256 + piece * 4) = make_float4(o[n][0], o[n][2], o[n + 1][0], o[n + 1][2]);
                    *reinterpret_cast<float4 *>(own + row1 * 256 + piece * 4) = make_float4(o[n][1], o[n][3], o[n + 1][1], o[n + 1][3]);
                }
        }
        __syncthreads();
        if (threadIdx.x < 8) {                         // one thread per row: the maximum, the warps' factors, the sum
            const int row = threadIdx.x;
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int k = 0; k < KG; k++) M = fmaxf(M, sm_m[k * 8 + row]);
#pragma unroll
            for (int k = 0; k < KG; k++) {
                const float r = sm_m[k * 8 + row], f = r == M ? 1.0f : ex2(r - M);
                L = fmaf(sm_l[k * 8 + row], f, L);
                sm_m[k * 8 + row] = f;
            }
            sm_t[row] = M; sm_t[8 + row] = L;
        }
        __syncthreads();
        const bool whole = seg_t0 == 0 && seg_n == sq.n_tiles;
        const size_t slot = (size_t)blockIdx.x + (size_t)w.s * p.kv_heads + w.h;
        const int in = min(KG, seg_n);                 // warps that had a tile
        for (int idx = threadIdx.x; idx < valid * 64; idx += D_THREADS) {
            const int row = idx >> 6, pc = idx & 63;
            const uint32_t piece = (uint32_t)pc ^ (uint32_t)((row >> 1) & 3);
            const float *src = reinterpret_cast<const float *>(smem) + row * 256 + piece * 4;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < KG; k++) {
                if (k < in) {
                    const float f = sm_m[k * 8 + row];
                    const float4 a = *reinterpret_cast<const float4 *>(src + k * (NS * ENTRY / 4));
                    acc.x = fmaf(a.x, f, acc.x); acc.y = fmaf(a.y, f, acc.y); acc.z = fmaf(a.z, f, acc.z); acc.w = fmaf(a.w, f, acc.w);
                }
            }
            const float M = sm_t[row], L = sm_t[8 + row];
            if (whole) {
                const int r = row / p.gqa;
                const float inv = 1.0f / L;
                store_out(p, sq, (size_t)r * p.q_heads + head0 + (row - r * p.gqa), pc * 4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
            } else {
                const size_t pi = slot * p.slot_rows + row;
                *reinterpret_cast<float4 *>(p.pacc + pi * 256 + pc * 4) = acc;
                if (pc == 0) *reinterpret_cast<float2 *>(p.pstat + pi * 2) = make_float2(M, L);
            }
        }
        T += seg_n;
        w.t = 0;                                          // the next segment, if any, begins the next group
        if (++w.h == p.kv_heads) { w.h = 0; w.s++; }
        fence_proxy_async();                              // the ring goes back to the copy engine
        __syncthreads();
    }
    if (*abort_flag)                                      // a wait gave up: copies of this CTA may still be under way
        for (int i = 0; i < 4096; i++) __nanosleep(10000);
}

// =======================================================================================
// attention, 9 to 32 query rows (a verify step)
// =======================================================================================
// NT tiles of eight query rows.  Two warps share a tile of 32 keys: each scores 16 of its keys against all rows (the K
// codes are widened once, however many rows there are) and each takes 128 dims of V for all 32 keys.  What they swap is
// the weights, through shared memory.  The running maximum is the pair's and lags: it moves only when a score exceeds it
// by more than 2^4 (the pair votes with the barrier that also guards the weights' buffer), so that most tiles need no
// reduction over the lanes and no rescaling; the weights reach 2^15 then, which fp16 holds.  Four tokens of 24 heads over
// 4 behind 32 K keys: 26.0 us, of which the 67 MB take 10.3.  What bounds it is the chain inside a tile (scores, vote,
// weights, swap, products: about 3 us, four or five tiles to a pair) and 12 us of launch, first loads, sums and merge.
constexpr float VF_LAG = 4.0f, VF_SHIFT = 11.0f;

template <int NT, bool F32>
struct VfCfg {
    static constexpr int WARPS = NT == 4 ? 8 : 12, PAIRS = WARPS / 2, THREADS = WARPS * 32;
    static constexpr int VS = F32 && NT == 3 ? 1 : 2, NS = 2 + VS;       // 4 KB slots of a warp: two for its part of K, VS for its part of V
    static constexpr int PX = NT * 32 * (F32 ? 16 : 8);         // weights of one warp's keys, as B fragments
    static constexpr int ROWS = NT * 8;
    static constexpr int OFF_Q = WARPS * NS * 4096;
    static constexpr int OFF_PX = OFF_Q + NT * (F32 ? 8192 : 4096);       // [pair][half]
    static constexpr int OFF_MX = OFF_PX + WARPS * PX;          // [warp][ROWS] maxima of a tile
    static constexpr int OFF_M = OFF_MX + WARPS * ROWS * 4;     // [pair][ROWS], then the pair's factor
    static constexpr int OFF_L = OFF_M + PAIRS * ROWS * 4;      // [warp][ROWS]
    static constexpr int OFF_T = OFF_L + WARPS * ROWS * 4;      // [2][ROWS] maximum and sum of all pairs
    static constexpr int OFF_SC = OFF_T + 2 * ROWS * 4;         // [ROWS]
    static constexpr int OFF_LIM = OFF_SC + ROWS * 4;           // [ROWS] last key of a row
    static constexpr int OFF_BAR = OFF_LIM + ROWS * 4;           // full[warp][slot], abort
    static constexpr int SMEM = OFF_BAR + WARPS * NS * 8 + 16;
    static_assert(SMEM <= 232448, "exceeds the 227 KB a CTA may use");
    static_assert(NT <= NS, "a warp's sums do not fit its slots");
};

template <int NT, bool F32>
__global__ void __launch_bounds__(VfCfg<NT, F32>::THREADS, 1) kv8_verify_kernel(const __grid_constant__ Kv8AttnParams p) {
    using Cfg = VfCfg<NT, F32>;
    constexpr int NS = Cfg::NS, VS = Cfg::VS, PAIRS = Cfg::PAIRS, ROWS = Cfg::ROWS;
    extern __shared__ __align__(1024) uint8_t smem[];
    float *sm_m = reinterpret_cast<float *>(smem + Cfg::OFF_M);
    float *sm_l = reinterpret_cast<float *>(smem + Cfg::OFF_L);
    float *sm_t = reinterpret_cast<float *>(smem + Cfg::OFF_T);
    float *sm_sc = reinterpret_cast<float *>(smem + Cfg::OFF_SC);
    int *sm_lim = reinterpret_cast<int *>(smem + Cfg::OFF_LIM);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + Cfg::OFF_BAR);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(full + Cfg::WARPS * NS);

    if (smem_u32(smem) & 1023u) {                    // swizzled boxes need 1024-byte alignment
        if (threadIdx.x == 0) report(p.status, QW_ST_BAD_SMEM);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pair = warp >> 1, half = warp & 1;
    const int g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) {
        for (int i = 0; i < Cfg::WARPS * NS; i++) mbar_init(&full[i], 1);
        *abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&p.maps[0]);
        tma_prefetch_desc(&p.maps[1]);
    }
    const int lo = p.share[blockIdx.x], hi = p.share[blockIdx.x + 1];
    Where w = locate(p, lo);
    {
        const Kv8AttnSeq &sq = p.seq[w.s];
#pragma unroll 1
        for (int i = warp; i < ROWS; i += Cfg::WARPS) prefetch_rows(sq.q, p.io, (size_t)w.h * p.gqa * 256, 256, sq.rows, p.gqa, p.q_heads, i, lane);
        // (the first tile only: with the second the merge kernel before this one waits longer than the loads gain)
        if (pair < min(sq.n_tiles - w.t, hi - lo)) warm_tile<16>(p, sq, w.h, w.t + pair, 16 * half, 128 * half, lane);
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_next();

    uint8_t *ring = smem + warp * NS * 4096;
    uint64_t *full_k = full + warp * NS, *full_v = full_k + 2;
    uint8_t *px = smem + Cfg::OFF_PX + pair * 2 * Cfg::PX;
    float *mx = reinterpret_cast<float *>(smem + Cfg::OFF_MX) + pair * 2 * ROWS;
    uint32_t done = 0;                               // tiles of this pair before the current segment

    for (int T = lo; T < hi;) {
        const Kv8AttnSeq &sq = p.seq[w.s];
        const int seg_t0 = w.t, seg_n = min(sq.n_tiles - w.t, hi - T);
        const int valid = sq.rows * p.gqa, head0 = w.h * p.gqa;
        const int n_keys = sq.base_pos + sq.rows;
        const int nt = pair < seg_n ? (seg_n - pair + PAIRS - 1) / PAIRS : 0;      // this pair's tiles

        // code rows of 32 tiles, one per lane, looked up two tiles ahead of their use; exponents of 32 tiles
        int win_k = 0, win_v = 0, win_e = 0;
        auto key_of = [&](int i) { return (seg_t0 + pair + i * PAIRS) * TILE; };
        auto rows_from = [&](int i0) {
            if (i0 + lane >= nt) return;
            win_k = tile_row(p, sq.ktab, w.h, key_of(i0 + lane)); win_v = tile_row(p, sq.vtab, w.h, key_of(i0 + lane));
        };
        auto exps_from = [&](int i0) {
            if (i0 + lane >= nt) return;
            const int b = key_of(i0 + lane) / BLK;
            const int ek = clamp_exp(sq.kexp[(size_t)w.h * p.exp_stride + b]), ev = clamp_exp(sq.vexp[(size_t)w.h * p.exp_stride + b]);
            win_e = (ek & 0xffff) | (ev << 16);
        };
        // lane 0: this warp's 16 keys x 256 dims of K, and 32 keys x 128 dims of V, of the pair's n-th tile
        auto load_k = [&](uint32_t n, int row) {
            uint8_t *dst = ring + (n & 1) * 4096;
            uint64_t *bar = &full_k[n & 1];
            mbar_expect_tx(bar, 4096);
            tma_load_2d(dst, &p.maps[sq.kmap], 0, row + 16 * half, bar);
            tma_load_2d(dst + 2048, &p.maps[sq.kmap], 128, row + 16 * half, bar);
        };
        auto load_v = [&](uint32_t n, int row) {
            const uint32_t sl = VS == 2 ? n & 1 : 0;
            uint8_t *dst = ring + (2 + sl) * 4096;
            mbar_expect_tx(&full_v[sl], 4096);
            tma_load_2d(dst, &p.maps[sq.vmap], 128 * half, row, &full_v[sl]);
            tma_load_2d(dst + 2048, &p.maps[sq.vmap], 128 * half, row + 16, &full_v[sl]);
        };
        constexpr int PER = (ROWS + Cfg::WARPS - 1) / Cfg::WARPS;
        RowRaw<F32> raw[PER];
#pragma unroll
        for (int u = 0; u < PER; u++) raw[u] = fetch_q<F32>(p, sq, head0, valid, warp + u * Cfg::WARPS, lane);
        // (only the first part of K is asked for at once: what is on its way to all SMs in front of the query rows holds them up)
        int k1 = 0, v1 = 0;
        if (nt > 0) {
            rows_from(0);
            exps_from(0);
            k1 = __shfl_sync(0xffffffffu, win_k, 1); v1 = __shfl_sync(0xffffffffu, win_v, 1);
            if (lane == 0) load_k(done, win_k);
        }
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int row = warp + u * Cfg::WARPS;
            next_rows(p, w, sq, seg_t0, seg_n, T, hi, row, lane);
            if (row < ROWS) stage_q<F32>(p, raw[u], row, lane, smem + Cfg::OFF_Q, sm_sc + row);
        }
        if (nt > 0 && lane == 0) {
            load_v(done, win_v);
            if (nt > 1) {
                load_k(done + 1, k1);
                if (VS == 2) load_v(done + 1, v1);
            }
        }
        if (threadIdx.x < ROWS) sm_lim[threadIdx.x] = (int)threadIdx.x < valid ? sq.base_pos + (int)threadIdx.x / p.gqa : n_keys - 1;
        __syncthreads();

        float o[NT][8][4];
        float l[NT][2], R[NT][2];                    // rows 8 n + 2 t and the one after it
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < 8; j++) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
            R[n][0] = R[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
        }
        const uint32_t q_base = smem_u32(smem + Cfg::OFF_Q) + lane * 16;
        const uint32_t tok = (uint32_t)(g ^ ((g & 1) << 2));         // this lane group's key of a block of eight

#pragma unroll 1
        for (int i = 0; i < nt; i++) {
            const int key0 = (seg_t0 + pair + i * PAIRS) * TILE;
            const uint32_t n_t = done + i;
            if (i > 0 && (i & 31) == 0) exps_from(i);
            const int ex = __shfl_sync(0xffffffffu, win_e, i & 31);
            constexpr int AHEAD_V = VS == 2 ? 2 : 1;
            int nv = __shfl_sync(0xffffffffu, win_v, (i + 1) & 31);
            if (((i + 2) & 31) == 0) rows_from(i + 2);
            const int nk = __shfl_sync(0xffffffffu, win_k, (i + 2) & 31);
            if (VS == 2) nv = __shfl_sync(0xffffffffu, win_v, (i + 2) & 31);
            const int ek = (int)(int16_t)(ex & 0xffff), ev = ex >> 16;

            // ---- S^T = K Q^T for this warp's 16 keys ----
            float s[NT][4], sl[NT][4];                 // (f32: the low parts have sums of their own, as in the decode kernel)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[n][c] = sl[n][c] = 0.0f;
            mbar_wait(&full_k[n_t & 1], (n_t >> 1) & 1, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
            {
                const uint32_t kb = smem_u32(ring + (n_t & 1) * 4096) + tok * 128;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t kw[2][4];                 // keys tok, tok + 8
#pragma unroll
                    for (int n = 0; n < 2; n++) lds128(kw[n], kb + (q >> 1) * 2048 + n * 1024 + ((((uint32_t)(4 * (q & 1) + t)) ^ tok) << 4));
#pragma unroll
                    for (int kk = 0; kk < 2; kk++) {
                        uint32_t b[NT][4];             // two k-steps of Q (f32: one, high and low)
                        if constexpr (!F32) {
#pragma unroll
                            for (int n = 0; n < NT; n++) lds128(b[n], q_base + n * 4096 + (q * 2 + kk) * 512);
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int k = kk * 2 + h;
                            if constexpr (F32) {
#pragma unroll
                                for (int n = 0; n < NT; n++) lds128(b[n], q_base + n * 8192 + (q * 4 + k) * 512);
                            }
                            const uint32_t a0 = f16x2_lo(kw[0][k]), a1 = f16x2_lo(kw[1][k]), a2 = f16x2_hi(kw[0][k]), a3 = f16x2_hi(kw[1][k]);
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                if constexpr (F32) {
                                    mma_f16(s[n], a0, a1, a2, a3, b[n][0], b[n][1]);
                                    mma_f16(sl[n], a0, a1, a2, a3, b[n][2], b[n][3]);
                                } else {
                                    mma_f16(s[n], a0, a1, a2, a3, b[n][2 * h], b[n][2 * h + 1]);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && i + 2 < nt) load_k(n_t + 2, nk);

            // ---- scores; does any exceed the running maximum by more than it may lag? ----
            const float fk = pow2f(ek), fv = (float)ev;
            const bool masked = key0 + TILE > sq.base_pos + 1;
            bool over = false;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float2 sc = *reinterpret_cast<const float2 *>(sm_sc + n * 8 + 2 * t);
#pragma unroll
                for (int c = 0; c < 4; c++) s[n][c] = fmaf(F32 ? s[n][c] + sl[n][c] : s[n][c], ((c & 1) ? sc.y : sc.x) * fk, fv);
                if (masked) {
                    const int2 lim = *reinterpret_cast<const int2 *>(sm_lim + n * 8 + 2 * t);
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (key0 + 16 * half + (c >> 1) * 8 + (int)tok > ((c & 1) ? lim.y : lim.x)) s[n][c] = -INFINITY;
                }
                over |= fmaxf(s[n][0], s[n][2]) > R[n][0] + VF_LAG || fmaxf(s[n][1], s[n][3]) > R[n][1] + VF_LAG;
            }
            uint32_t move;
            asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %2, 0;\n\tbarrier.cta.red.or.pred b, %1, 64, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
                         : "=r"(move) : "r"(1 + pair), "r"((uint32_t)over) : "memory");
            if (move) {
                float x[NT][2];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    x[n][0] = fmaxf(s[n][0], s[n][2]); x[n][1] = fmaxf(s[n][1], s[n][3]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        x[n][0] = fmaxf(x[n][0], __shfl_xor_sync(0xffffffffu, x[n][0], d));
                        x[n][1] = fmaxf(x[n][1], __shfl_xor_sync(0xffffffffu, x[n][1], d));
                    }
                    if (g == 0) *reinterpret_cast<float2 *>(mx + half * ROWS + n * 8 + 2 * t) = make_float2(x[n][0], x[n][1]);
                }
                asm volatile("barrier.cta.sync %0, 64;" ::"r"(1 + pair) : "memory");
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const float2 y = *reinterpret_cast<const float2 *>(mx + (half ^ 1) * ROWS + n * 8 + 2 * t);
                    const float n0 = fmaxf(R[n][0], fmaxf(x[n][0], y.x)), n1 = fmaxf(R[n][1], fmaxf(x[n][1], y.y));
                    const float f0 = R[n][0] == n0 ? 1.0f : ex2(R[n][0] - n0), f1 = R[n][1] == n1 ? 1.0f : ex2(R[n][1] - n1);
                    l[n][0] *= f0; l[n][1] *= f1;
#pragma unroll
                    for (int j = 0; j < 8; j++) { o[n][j][0] *= f0; o[n][j][1] *= f1; o[n][j][2] *= f0; o[n][j][3] *= f1; }
                    R[n][0] = n0; R[n][1] = n1;
                }
            }

            // ---- weights of this warp's keys, to the other warp as well ----
            const float iv = pow2f(-ev);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float b0 = (R[n][0] == -INFINITY ? 0.0f : R[n][0]) - VF_SHIFT, b1 = (R[n][1] == -INFINITY ? 0.0f : R[n][1]) - VF_SHIFT;
                uint32_t pb[2], pl[2];
                float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float w0 = ex2(s[n][2 * c] - b0), w1 = ex2(s[n][2 * c + 1] - b1);
                    a0 += w0; a1 += w1;
                    const uint32_t hi = pack_f16(w0, w1);
                    pb[c] = movm(hi);
                    if constexpr (F32) {
                        const float2 h = h2f2(hi);
                        pl[c] = movm(pack_f16(w0 - h.x, w1 - h.y));
                    }
                }
                l[n][0] = fmaf(a0, iv, l[n][0]); l[n][1] = fmaf(a1, iv, l[n][1]);
                if constexpr (F32) reinterpret_cast<uint4 *>(px + half * Cfg::PX)[n * 32 + lane] = make_uint4(pb[0], pb[1], pl[0], pl[1]);
                else reinterpret_cast<uint2 *>(px + half * Cfg::PX)[n * 32 + lane] = make_uint2(pb[0], pb[1]);
            }
            asm volatile("barrier.cta.sync %0, 64;" ::"r"(1 + pair) : "memory");

            // ---- O^T += V^T P^T: row g of tile j is dim 128 half + 16 g + 2 j, row g + 8 the dim after it ----
            const uint32_t vsl = VS == 2 ? n_t & 1 : 0;
            mbar_wait(&full_v[vsl], VS == 2 ? (n_t >> 1) & 1 : n_t & 1, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
            uint8_t *vs = ring + (2 + vsl) * 4096;
            if (key0 + TILE > n_keys) {                // rows past the last key may hold anything
                for (int off = (n_keys - key0) * 128 + lane * 16; off < TILE * 128; off += 512) *reinterpret_cast<uint4 *>(vs + off) = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
                __syncwarp();
            }
            const uint32_t vb = smem_u32(vs);
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {           // the keys of either warp
                uint32_t b[NT][F32 ? 4 : 2];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    if constexpr (F32) {
                        const uint4 x = reinterpret_cast<const uint4 *>(px + kk * Cfg::PX)[n * 32 + lane];
                        b[n][0] = x.x; b[n][1] = x.y; b[n][2] = x.z; b[n][3] = x.w;
                    } else {
                        const uint2 x = reinterpret_cast<const uint2 *>(px + kk * Cfg::PX)[n * 32 + lane];
                        b[n][0] = x.x; b[n][1] = x.y;
                    }
                }
                const uint32_t ta = 16 * kk + 2 * t, tb = 16 * kk + ((2 * t + 1) ^ 4);
                uint32_t v[4][4];                      // keys ta, tb, ta + 8, tb + 8
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t tk = ((c & 1) ? tb : ta) + (c >> 1) * 8;
                    lds128(v[c], vb + tk * 128 + (((uint32_t)g ^ (tk & 7)) << 4));
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t p0 = __byte_perm(v[0][k], v[1][k], 0x5140), p1 = __byte_perm(v[0][k], v[1][k], 0x7362);
                    const uint32_t r0 = __byte_perm(v[2][k], v[3][k], 0x5140), r1 = __byte_perm(v[2][k], v[3][k], 0x7362);
                    const uint32_t c0 = f16x2_lo(p0), c1 = f16x2_hi(p0), c2 = f16x2_lo(r0), c3 = f16x2_hi(r0);
                    const uint32_t d0 = f16x2_lo(p1), d1 = f16x2_hi(p1), d2 = f16x2_lo(r1), d3 = f16x2_hi(r1);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        mma_f16(o[n][2 * k], c0, c1, c2, c3, b[n][0], b[n][1]);
                        mma_f16(o[n][2 * k + 1], d0, d1, d2, d3, b[n][0], b[n][1]);
                        if constexpr (F32) {
                            mma_f16(o[n][2 * k], c0, c1, c2, c3, b[n][2], b[n][3]);
                            mma_f16(o[n][2 * k + 1], d0, d1, d2, d3, b[n][2], b[n][3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && i + AHEAD_V < nt) load_v(n_t + AHEAD_V, nv);
        }
        done += nt;

        // ---- segment end: every warp puts its 128 dims of all rows into its slots, and all threads add them up ----
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], d);
                if (g == 0) {
                    if (half == 0) sm_m[pair * ROWS + n * 8 + 2 * t + c] = R[n][c];
                    sm_l[warp * ROWS + n * 8 + 2 * t + c] = l[n][c];
                }
            }
        }
        if (nt > 0) {
            // piece c (four dims) of a row sits at c ^ ((row >> 1) & 3), which spreads a phase's eight lanes over the banks
            float *own = reinterpret_cast<float *>(ring);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t piece = (uint32_t)(g * 4 + e) ^ (uint32_t)t;
                    const int row = n * 8 + 2 * t;
                    *reinterpret_cast<float4 *>(own + row * 128 + piece * 4) = make_float4(o[n][2 * e][0], o[n][2 * e][2], o[n][2 * e + 1][0], o[n][2 * e + 1][2]);
                    *reinterpret_cast<float4 *>(own + (row + 1) * 128 + piece * 4) = make_float4(o[n][2 * e][1], o[n][2 * e][3], o[n][2 * e + 1][1], o[n][2 * e + 1][3]);
                }
        }
        __syncthreads();
        if (threadIdx.x < ROWS) {                      // one thread per row: the maximum, the pairs' factors, the sum
            const int row = threadIdx.x;
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int k = 0; k < PAIRS; k++) M = fmaxf(M, sm_m[k * ROWS + row]);
#pragma unroll
            for (int k = 0; k < PAIRS; k++) {
                const float r = sm_m[k * ROWS + row], f = r == M ? 1.0f : ex2(r - M);
                L = fmaf(sm_l[2 * k * ROWS + row] + sm_l[(2 * k + 1) * ROWS + row], f, L);
                sm_m[k * ROWS + row] = f;
            }
            sm_t[row] = M; sm_t[ROWS + row] = L;
        }
        __syncthreads();
        const bool whole = seg_t0 == 0 && seg_n == sq.n_tiles;
        const size_t slot = (size_t)blockIdx.x + (size_t)w.s * p.kv_heads + w.h;
        const int in = min(PAIRS, seg_n);              // pairs that had a tile
        for (int idx = threadIdx.x; idx < valid * 64; idx += Cfg::THREADS) {
            const int row = idx >> 6, pc = idx & 63;
            const uint32_t piece = (uint32_t)(pc & 31) ^ (uint32_t)((row >> 1) & 3);
            const float *src = reinterpret_cast<const float *>(smem + (pc >> 5) * NS * 4096) + row * 128 + piece * 4;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < PAIRS; k++) {
                if (k < in) {
                    const float f = sm_m[k * ROWS + row];
                    const float4 a = *reinterpret_cast<const float4 *>(src + (size_t)k * 2 * NS * 1024);
                    acc.x = fmaf(a.x, f, acc.x); acc.y = fmaf(a.y, f, acc.y); acc.z = fmaf(a.z, f, acc.z); acc.w = fmaf(a.w, f, acc.w);
                }
            }
            if (whole) {
                const int r = row / p.gqa;
                const float inv = 1.0f / sm_t[ROWS + row];
                store_out(p, sq, (size_t)r * p.q_heads + head0 + (row - r * p.gqa), pc * 4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
            } else {
                const size_t pi = slot * p.slot_rows + row;
                *reinterpret_cast<float4 *>(p.pacc + pi * 256 + pc * 4) = acc;
                if (pc == 0) *reinterpret_cast<float2 *>(p.pstat + pi * 2) = make_float2(sm_t[row], sm_t[ROWS + row]);
            }
        }
        T += seg_n;
        w.t = 0;                                          // the next segment, if any, begins the next group
        if (++w.h == p.kv_heads) { w.h = 0; w.s++; }
        fence_proxy_async();                              // the ring goes back to the copy engine
        __syncthreads();
    }
    if (*abort_flag)                                      // a wait gave up: copies of this CTA may still be under way
        for (int i = 0; i < 4096; i++) __nanosleep(10000);
}

// Partials of a cut group: one block per (group, row).  (A kernel of its own: it starts under the attention kernel's tail,
// and the next call's attention under its own.  Added up by the last CTA of a group instead, behind a counter, a decode
// step over 4 K keys took 12.2 us against 8.9.)  Slices of 64 threads x four dims take every MG_SLICES-th
// partial each, ten loads in flight, asked for before the weights are known: one trip to L2 for up to 40 partials
// (four slices: many groups, few partials each) or 160 (sixteen: few groups, cut over most of the SMs).
constexpr int MG_FLY = 10;
template <int MG_SLICES>
__global__ void __launch_bounds__(MG_SLICES * 64) kv8_merge_kernel(const __grid_constant__ Kv8AttnParams p, int max_valid) {
    __shared__ float w_s[256];
    __shared__ float red_s[2][8];
    __shared__ __align__(16) float acc_s[MG_SLICES][256];
    pdl_launch_next();
    const int gi = blockIdx.x / max_valid, row = blockIdx.x - gi * max_valid;
    const int s = gi / p.kv_heads, h = gi - s * p.kv_heads;
    const Kv8AttnSeq &sq = p.seq[s];
    const int G0 = sq.cum_tiles + h * sq.n_tiles, c0 = share_of(p, G0), parts = share_of(p, G0 + sq.n_tiles - 1) - c0 + 1;
    pdl_wait();
    if (row >= sq.rows * p.gqa || parts == 1) return;     // (a group of one part was written whole)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int slice = tid >> 6, d4 = (tid & 63) * 4;
    const size_t pi0 = (size_t)(c0 + gi) * p.slot_rows + row;
    const float *base = p.pacc + pi0 * 256 + d4;
    const size_t step = (size_t)p.slot_rows * 256;
    float4 a[MG_FLY];
#pragma unroll
    for (int u = 0; u < MG_FLY; u++) {
        const int q = slice + MG_SLICES * u;
        a[u] = q < parts ? *reinterpret_cast<const float4 *>(base + (size_t)q * step) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mq = -INFINITY, lq = 0.0f;
    if (tid < 256) {                                      // (parts <= CTAs <= 256)
        if (tid < parts) {
            const float2 st = *reinterpret_cast<const float2 *>(p.pstat + (pi0 + (size_t)tid * p.slot_rows) * 2);
            mq = st.x; lq = st.y;
        }
        const float m = warp_max(mq);
        if (lane == 0) red_s[0][warp] = m;
    }
    __syncthreads();
    float m = red_s[0][0];
#pragma unroll
    for (int i = 1; i < 8; i++) m = fmaxf(m, red_s[0][i]);
    if (tid < 256) {
        const float wq = mq == m ? 1.0f : ex2(mq - m);
        w_s[tid] = wq;
        const float d = warp_sum(tid < parts ? lq * wq : 0.0f);
        if (lane == 0) red_s[1][warp] = d;
    }
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < MG_FLY; u++) {
        const int q = slice + MG_SLICES * u;
        const float f = q < parts ? w_s[q] : 0.0f;
        acc.x = fmaf(a[u].x, f, acc.x); acc.y = fmaf(a[u].y, f, acc.y); acc.z = fmaf(a[u].z, f, acc.z); acc.w = fmaf(a[u].w, f, acc.w);
    }
    for (int q = slice + MG_SLICES * MG_FLY; q < parts; q += MG_SLICES) {
        const float4 b = *reinterpret_cast<const float4 *>(base + (size_t)q * step);
        const float f = w_s[q];
        acc.x = fmaf(b.x, f, acc.x); acc.y = fmaf(b.y, f, acc.y); acc.z = fmaf(b.z, f, acc.z); acc.w = fmaf(b.w, f, acc.w);
    }
    *reinterpret_cast<float4 *>(&acc_s[slice][d4]) = acc;
    __syncthreads();
    if (slice > 0) return;
    float den = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) den += red_s[1][i];
#pragma unroll
    for (int i = 1; i < MG_SLICES; i++) {
        const float4 b = *reinterpret_cast<const float4 *>(&acc_s[i][d4]);
        acc.x += b.x; acc.y += b.y; acc.z += b.z; acc.w += b.w;
    }
    const int r = row / p.gqa;
    const float inv = 1.0f / den;
    store_out(p, sq, (size_t)r * p.q_heads + h * p.gqa + (row - r * p.gqa), d4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
}

void pdl_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute &attr, dim3 grid, unsigned block, size_t smem, cudaStream_t s) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg = cudaLaunchConfig_t();
    cfg.gridDim = grid; cfg.blockDim = dim3(block); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cfg.attrs = &attr; cfg.numAttrs = g_tune_pdl ? 1 : 0;
}

template <bool F32>
void launch_decode_t(cudaStream_t s, const Kv8AttnParams &p) {
    static bool configured[64] = {false};      // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        cudaFuncSetAttribute(kv8_decode_kernel<F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, D_SMEM);
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    pdl_config(cfg, attr, dim3((unsigned)p.n_cta), D_THREADS, D_SMEM, s);
    cudaLaunchKernelEx(&cfg, kv8_decode_kernel<F32>, p);
    g_launches++;
}

template <int NT, bool F32>
void launch_verify_t(cudaStream_t s, const Kv8AttnParams &p) {
    using Cfg = VfCfg<NT, F32>;
    static bool configured[64] = {false};      // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        cudaFuncSetAttribute(kv8_verify_kernel<NT, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    pdl_config(cfg, attr, dim3((unsigned)p.n_cta), Cfg::THREADS, Cfg::SMEM, s);
    cudaLaunchKernelEx(&cfg, kv8_verify_kernel<NT, F32>, p);
    g_launches++;
}

}  // namespace

void launch_kv8_write(cudaStream_t s, const Kv8WriteParams &p) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    pdl_config(cfg, attr, dim3((unsigned)p.max_blocks, (unsigned)p.kv_heads * 2, (unsigned)p.n_seq), WR_THREADS, 0, s);
    if (p.io == DT_BF16) cudaLaunchKernelEx(&cfg, kv8_write_kernel<__nv_bfloat16>, p);
    else cudaLaunchKernelEx(&cfg, kv8_write_kernel<float>, p);
    g_launches++;
}

template <typename T, int RD_ROWS>
static void launch_read_t(cudaStream_t s, void *dst, const Kv8Layer &c, int kv_heads, int pos0, int n) {
    constexpr int rows = RD_THREADS / 32 * RD_ROWS;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    pdl_config(cfg, attr, dim3((unsigned)((n + rows - 1) / rows), (unsigned)kv_heads), RD_THREADS, 0, s);
    cudaLaunchKernelEx(&cfg, kv8_read_kernel<T, RD_ROWS>, reinterpret_cast<T *>(dst), c, pos0, n);
    g_launches++;
}
void launch_kv8_read(cudaStream_t s, void *dst, int io, const Kv8Layer &c, int kv_heads, int pos0, int n) {
    const bool many = (int64_t)n * kv_heads >= 65536;        // several rounds of CTAs either way (measured: see the kernel)
    if (io == DT_BF16) { if (many) launch_read_t<__nv_bfloat16, 4>(s, dst, c, kv_heads, pos0, n); else launch_read_t<__nv_bfloat16, 2>(s, dst, c, kv_heads, pos0, n); }
    else { if (many) launch_read_t<float, 4>(s, dst, c, kv_heads, pos0, n); else launch_read_t<float, 2>(s, dst, c, kv_heads, pos0, n); }
}

void kv8_attn_plan(Kv8AttnParams &p) {
    int cum = 0, valid = 0;
    for (int i = 0; i < p.n_seq; i++) {
        Kv8AttnSeq &s = p.seq[i];
        s.n_tiles = (s.base_pos + s.rows + TILE - 1) / TILE;
        s.cum_tiles = cum;
        cum += s.n_tiles * p.kv_heads;
        valid = std::max(valid, s.rows * p.gqa);
    }
    p.total_tiles = cum;
    p.n_cta = std::min(std::min(sm_count(), 256), cum);
    p.slot_rows = valid;
    // Shares of equal cost: a share that begins a group pays that segment's first loads and its sum over the warps
    // on top of its tiles, SEG_COST tile times.  So every group is given that many virtual tiles in front, the virtual
    // line is cut evenly, and a cut among the virtual tiles moves to the group's first real one.
    const int groups = p.n_seq * p.kv_heads;
    const int64_t v_total = (int64_t)cum + (int64_t)SEG_COST * groups;
    int s = 0, h = 0, t0 = 0;                                // group (s, h) and its first real tile
    int64_t v0 = 0, v = 0, rest = 0;                         // its virtual start; v = floor(v_total * c / n_cta)
    const int64_t step = v_total / p.n_cta, more = v_total % p.n_cta;
    for (int c = 0; c < p.n_cta; c++) {
        while (v >= v0 + SEG_COST + p.seq[s].n_tiles) {
            v0 += SEG_COST + p.seq[s].n_tiles;
            t0 += p.seq[s].n_tiles;
            if (++h == p.kv_heads) { h = 0; s++; }
        }
        p.share[c] = t0 + (int)std::max<int64_t>(0, v - v0 - SEG_COST);
        v += step;
        rest += more;
        if (rest >= p.n_cta) { rest -= p.n_cta; v++; }
    }
    p.share[p.n_cta] = cum;
}

// Partials of the group that has the most (0: no group is cut).
static int most_parts(const Kv8AttnParams &p) {
    int parts = 0;
    for (int i = 0; i < p.n_seq; i++)
        for (int h = 0; h < p.kv_heads; h++) {
            const int g0 = p.seq[i].cum_tiles + h * p.seq[i].n_tiles;
            parts = std::max(parts, share_of(p, g0 + p.seq[i].n_tiles - 1) - share_of(p, g0));
        }
    return parts ? parts + 1 : 0;
}

size_t kv8_attn_scratch_bytes(const Kv8AttnParams &p) {
    return ((size_t)p.n_cta + (size_t)p.n_seq * p.kv_heads) * p.slot_rows * 258 * sizeof(float);
}

void launch_kv8_attn(cudaStream_t s, Kv8AttnParams &p, int max_rows, void *scratch) {
    const size_t slots = (size_t)p.n_cta + (size_t)p.n_seq * p.kv_heads;
    p.pacc = reinterpret_cast<float *>(scratch);
    p.pstat = p.pacc + slots * p.slot_rows * 256;
    const int valid = max_rows * p.gqa, nt = (valid + 7) / 8;
    const bool f32 = p.io == DT_F32;
    if (nt <= 1) { if (f32) launch_decode_t<true>(s, p); else launch_decode_t<false>(s, p); }
    else if (nt == 2) { if (f32) launch_verify_t<2, true>(s, p); else launch_verify_t<2, false>(s, p); }
    else if (nt == 3) { if (f32) launch_verify_t<3, true>(s, p); else launch_verify_t<3, false>(s, p); }
    else { if (f32) launch_verify_t<4, true>(s, p); else launch_verify_t<4, false>(s, p); }
    const int parts = most_parts(p);
    if (!parts) return;                        // every group was written whole
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    const bool few = parts <= 4 * MG_FLY;
    pdl_config(cfg, attr, dim3((unsigned)(p.n_seq * p.kv_heads * valid)), few ? 256 : 1024, 0, s);
    if (few) cudaLaunchKernelEx(&cfg, kv8_merge_kernel<4>, p, valid);
    else cudaLaunchKernelEx(&cfg, kv8_merge_kernel<16>, p, valid);
    g_launches++;
}

}  // namespace qw
