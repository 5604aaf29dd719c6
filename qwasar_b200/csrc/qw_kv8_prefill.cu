// Attention over the 8-bit cache for many query rows: tcgen05 tensor cores, accumulators in tensor memory (sm_100a).
//
// One CTA per (tile of 128 query rows, kv head, share of the keys).  A tile packs R = 128 / grouping rows of the call
// with all query heads of the kv head: tile row i is row i / grouping, head i % grouping, so K and V are read once for
// the whole group.  128 keys per step:
//
//   warp 9       TMA: the Q tile, then K codes (two stages of 128 keys x 256 dims, 32 KB)
//   warps 12-15  V: codes from memory into registers, 64 keys ahead, widened to fp16 (exact) into three 32 KB stages of
//                64 keys; keys past the last one are zeros
//   warp 8       one thread issues  S  = Q K_j^T   (kind::f8f6f4: the K codes enter as they lie in the cache)
//   warp 11      one thread issues  O += P_j V_j   (kind::f16, P in tensor memory)
//   warps 0-7    softmax: two threads per tile row, 64 keys of every step each -- one block of the cache, so one
//                exponent of K and one of V per thread and step
//
// Q in 8 bits.  A bf16 number has eight significant bits, an e4m3 number four: q = high + low, both e4m3, exactly as
// long as neither leaves e4m3's range (below 2^-17 of the row's largest element the low part is rounded).  So S is two
// 8-bit products instead of one 16-bit product, at the same tensor time, and K needs no widening.  P is not cut this
// way: its small weights reach far below e4m3's range.  It is fp16, scaled by 2^7 (weights up to 2^15 while the
// running maximum lags by up to 2^8, down to 2^-31 of the maximum), and V is widened to match.
//
// Exponents: with t = scale * log2(e) * 2^(eq + ek) * s + ev and m the running maximum of t, w = 2^(t - m) weighs the V
// codes and l = sum w 2^-ev is the denominator, as in the split kernels of qw_kv8.cu.
//
// TMEM columns (512): O [0,256) fp32 | Q high [256,320) four dims a column | P [320,384) fp16 pairs | S [384,512) fp32.
// With few tiles the keys are cut into shares, so that all SMs have work; a share leaves (m, l, O) per tile row, and
// kv8_prefill_merge_kernel adds them up.  Every wait is bounded; tensor memory is always released.
//
// A step's products take about 2048 clocks of the tensor core; the softmax chain of a step (S out of tensor memory, maximum
// over 128 keys, 64 exponentials a thread, P back) takes about 2800 and is what bounds it, and tensor memory is full with
// one tile (O, Q, P and S are its 512 columns), so that little else runs under it.  Prompt of 4096 tokens, 16 heads over 4:
// 138 us, 1.0 PFLOP/s of 2 x 2 x 256 operations per visible pair; 499 tokens of 24 heads behind 16 K: 177 us, 1.1.
#include "qw_kernels.h"
#include <algorithm>
#include <cuda_fp16.h>

namespace qw {

namespace {

constexpr int BM = 128, BN = 128;
constexpr int K_BYTES = BN * 256, KBOX = BN * 128;    // K stage; 128 dims of it
constexpr int V_BYTES = 64 * 512, VBOX = 64 * 128;    // V fp16 of 64 keys; 64 dims of them
constexpr int V_ST = 3;
constexpr int IO_BOX = BM * 128;
constexpr int OFF_K = 0, OFF_V = 2 * K_BYTES, OFF_QLO = OFF_V + V_ST * V_BYTES;
constexpr int OFF_BAR = OFF_QLO + 2 * IO_BOX;
constexpr int OFF_STAGE_Q = OFF_V, OFF_STAGE_IO = OFF_K;      // Q tile (4 boxes bf16); gate / output (4 boxes), partial sums (8 boxes)
static_assert(OFF_V == 4 * IO_BOX && V_ST * V_BYTES >= 4 * IO_BOX, "a share's sums take the K and the V stages");
constexpr int COL_O = 0, COL_Q = 256, COL_P = 320, COL_S = 384;
constexpr int OFF_XCH = OFF_BAR + 256;                        // row maxima / sums passed between the two softmax halves
constexpr int SMEM_BYTES = OFF_XCH + 2 * 2 * BM * 4;
static_assert(SMEM_BYTES <= 232448, "exceeds the 227 KB a CTA may use");
constexpr int THREADS = 16 * 32;
constexpr int W_MMA = 8, W_K = 9, W_PV = 11, W_CV = 12;       // (warp 10: none)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG_BIG = -1.0e30f;
constexpr float RESCALE_AT = 8.0f, P_SHIFT = 7.0f;

enum Bar { Q_READY = 0, Q_FULL, G_FULL, K_FULL0, K_FULL1, K_FREE0, K_FREE1, V_FULL0, V_FULL1, V_FULL2, V_FREE0, V_FREE1, V_FREE2,
           S_READY, S_FREE, P_READY, PV_DONE, PV_ISSUED0, PV_ISSUED1, N_BARS };

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int clamp_exp(int byte) { return min(max(byte - 127, QW_KV8_E_MIN), QW_KV8_E_MAX); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t e4m3x2_of_f16(uint32_t v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(v));
    return r;
}
// a * sigmoid(g), b * sigmoid(h): two exponentials and one reciprocal (the unit that works them out delivers 16 a clock,
// and the output tile has 32 768 elements).  Gates below -43 count as -43: 2e-19.  A NaN stays in its own element.
__device__ __forceinline__ void gate2(float &a, float &b, float g, float h) {
    const float u = 1.0f + __expf(-fmaxf(g, -43.0f)), v = 1.0f + __expf(-fmaxf(h, -43.0f));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(u * v));
    a = g == g ? a * (r * v) : g;
    b = h == h ? b * (r * u) : h;
}
__device__ __forceinline__ uint32_t f16x2_of(uint32_t codes16) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes16));
    return r;
}

// ---- tcgen05 ------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], fp16
__device__ __forceinline__ void mma_ts_f16(bool acc, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 bd;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b64 bd, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %4, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
// the same with 8-bit operands, A in tensor memory or in shared memory
__device__ __forceinline__ void mma_ts_f8(bool acc, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 bd;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b64 bd, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], bd, %4, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void mma_ss_f8(bool acc, uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 ad, bd;\n\tsetp.ne.u32 p, %6, 0;\n\tmov.b64 ad, {%1, %2};\n\tmov.b64 bd, {%3, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], ad, bd, %5, p;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
          "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t addr, const uint32_t (&r)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor halves, SWIZZLE_128B, version 1 (see qw_prefill.cu); instruction descriptor with fp32
// accumulation and type code 0 for A and B: e4m3 in kind::f8f6f4, fp16 in kind::f16.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo_bytes) { return ((addr >> 4) & 0x3FFF) | (((lbo_bytes >> 4) & 0x3FFF) << 16); }
__device__ __forceinline__ constexpr uint32_t desc_hi(uint32_t sbo_bytes) { return ((sbo_bytes >> 4) & 0x3FFF) | (1u << 14) | (2u << 29); }
__device__ __forceinline__ constexpr uint32_t instr_desc(int m, int n, int b_mn_major) {
    return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, int32_t x, int32_t y, int32_t z, const void *src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void prefetch_3d(const CUtensorMap *map, int32_t x, int32_t y, int32_t z) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(map), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void bulk_store(void *dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
}

// Q of one thread: 128 dims (half wg) of tile row row_l, from the staged bf16 tile to the two e4m3 parts -- the high one in
// tensor memory, the low one in shared memory.  Returns scale * log2(e) * the row's power of two.  (A function of its own,
// not inlined: together with it the compiler orders the softmax loop 3 to 8 % slower.)
__device__ __noinline__ float stage_q(const Kv8PrefillParams &p, uint8_t *smem, uint64_t *bars, volatile int *abort_flag, float *xch, uint32_t t_q, int wg,
                                      int row_l, bool in_tile, uint32_t lane_base, int lane) {
    const uint32_t sw = row_l & 7;
    // this thread's 128 dims of its row: largest magnitude (with the other half's), then the two e4m3 parts
    const uint8_t *q_row = smem + OFF_STAGE_Q + 2 * wg * IO_BOX + row_l * 128;
    mbar_wait(&bars[Q_FULL], 0, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
    // (held in registers: read again between the stores below, each piece would wait for the one before it)
    uint4 x[16];
    uint32_t big = 0;                                          // magnitudes of bf16 order like their bits
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = *reinterpret_cast<const uint4 *>(q_row + (e >> 3) * IO_BOX + (((e & 7) ^ sw) << 4));
#pragma unroll
    for (int e = 0; e < 16; e++)
        big = __vmaxu2(__vmaxu2(big, x[e].x & 0x7fff7fffu), __vmaxu2(x[e].y & 0x7fff7fffu, __vmaxu2(x[e].z & 0x7fff7fffu, x[e].w & 0x7fff7fffu)));
    float mx = __uint_as_float(max(big & 0xffff0000u, big << 16));
    xch[wg * BM + row_l] = mx;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    mx = in_tile ? fmaxf(mx, xch[(wg ^ 1) * BM + row_l]) : 0.0f;
    const int k = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 100);     // scaled below 2^8
    const float f = in_tile ? pow2f(7 - k) : 0.0f;
    const float sc_row = fabsf(p.scale) * LOG2E * pow2f(k - 7);
    const float fs = p.scale < 0.0f ? -f : f;
    uint8_t *lo_row = smem + OFF_QLO + wg * IO_BOX + row_l * 128;
#pragma unroll
    for (int e = 0; e < 8; e++) {                              // 16 dims: four columns of high parts, a piece of low parts
        uint32_t hi4[4], lo4[4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t xw[4] = {x[2 * e + h].x, x[2 * e + h].y, x[2 * e + h].z, x[2 * e + h].w};
            uint32_t hc[4], lc[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // (eight significant bits fit fp16, so the difference to the high part is exact there)
                const float a0 = in_tile ? __uint_as_float(xw[i] << 16) * fs : 0.0f, a1 = in_tile ? __uint_as_float(xw[i] & 0xffff0000u) * fs : 0.0f;
                const uint32_t a = pack_f16(a0, a1);
                hc[i] = e4m3x2_of_f16(a);
                const uint32_t w = f16x2_of(hc[i]);
                const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&w));
                lc[i] = e4m3x2_of_f16(*reinterpret_cast<const uint32_t *>(&d));
            }
            hi4[h * 2] = hc[0] | (hc[1] << 16); hi4[h * 2 + 1] = hc[2] | (hc[3] << 16);
            lo4[h * 2] = lc[0] | (lc[1] << 16); lo4[h * 2 + 1] = lc[2] | (lc[3] << 16);
        }
        *reinterpret_cast<uint4 *>(lo_row + ((e ^ sw) << 4)) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
        tmem_st4(t_q + lane_base + wg * 32 + e * 4, hi4);
    }
    fence_proxy_async();                                       // the low parts are read by the tensor core
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[Q_READY]);
    asm volatile("bar.sync 1, 256;" ::: "memory");             // (xch is written again below)
    return sc_row;
}

// The 128 softmax threads of half wg, with what they wrote to shared memory in view of the copy engine.
__device__ __forceinline__ void half_sync(int wg) {
    fence_proxy_async();
    if (wg == 0) asm volatile("bar.sync 2, 128;" ::: "memory");
    else asm volatile("bar.sync 3, 128;" ::: "memory");
}

// The finished tile of one thread: 128 dims of its row, divided by the denominator, gated, into the output boxes.
__device__ __noinline__ void finish_tile(const Kv8PrefillParams &p, uint8_t *smem, uint64_t *bars, volatile int *abort_flag, uint32_t t_o, int wg, int row_l,
                                         uint32_t lane_base, bool elected, bool gated, float l, int kvh, int r0) {
    const uint32_t sw = row_l & 7;
    uint8_t *io_row = smem + OFF_STAGE_IO + row_l * 128;
    uint32_t v[32];
    if (gated) mbar_wait(&bars[G_FULL], 0, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
    const float inv = 1.0f / l;
#pragma unroll 1
    for (int c = 4 * wg; c < 4 * wg + 4; c++) {        // 32 outputs = 64 bytes = half a box row
        tmem_ld32(t_o + lane_base + c * 32, v);
        uint4 *bx = reinterpret_cast<uint4 *>(io_row + (c >> 1) * IO_BOX);
        uint4 gt[4];
#pragma unroll
        for (int k = 0; k < 4; k++) gt[k] = gated ? bx[((c & 1) * 4 + k) ^ sw] : make_uint4(0, 0, 0, 0);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = __uint_as_float(v[k * 8 + e]) * inv;
            if (gated) {
                const uint32_t gw[4] = {gt[k].x, gt[k].y, gt[k].z, gt[k].w};
#pragma unroll
                for (int e = 0; e < 4; e++) gate2(o[2 * e], o[2 * e + 1], __uint_as_float(gw[e] << 16), __uint_as_float(gw[e] & 0xffff0000u));
            }
            bx[((c & 1) * 4 + k) ^ sw] = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
        }
        if (c & 1) {
            half_sync(wg);
            if (elected) { tma_store_3d(&p.omap, (c >> 1) * 64, kvh * p.gqa, r0, smem + OFF_STAGE_IO + (c >> 1) * IO_BOX); tma_store_commit(); }
        }
    }
}

__global__ void __launch_bounds__(THREADS, 1) kv8_prefill_kernel(const __grid_constant__ Kv8PrefillParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {                      // swizzled boxes need 1024-byte alignment
        if (threadIdx.x == 0) report(p.status, QW_ST_BAD_SMEM);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + OFF_BAR);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + N_BARS);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // heaviest tiles (latest rows) first; consecutive CTAs are the shares of one tile
    const int item = blockIdx.x, part = item % p.splits;
    const int kvh = (item / p.splits) % p.kv_heads;
    const int qt = p.n_q_tiles - 1 - item / (p.splits * p.kv_heads);
    const int r0 = qt * p.tile_rows;                               // first row of the call in this tile
    const int n_keys = p.base_pos + p.rows;
    const int k_end = min(n_keys, p.base_pos + r0 + p.tile_rows);   // keys any row of this tile may read
    const int steps = (k_end + BN - 1) / BN;
    const int j0 = (int)((int64_t)steps * part / p.splits), n_t = (int)((int64_t)steps * (part + 1) / p.splits) - j0;
    const bool whole = p.splits == 1;
    const bool gated = whole && p.gated;

    pdl_wait();
    pdl_launch_next();
    float2 *stat = reinterpret_cast<float2 *>(p.pstat) + (size_t)item * BM;
    if (n_t == 0) {                                    // a share without a step: an empty partial
        if (threadIdx.x < BM) stat[threadIdx.x] = make_float2(NEG_BIG, 0.0f);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < N_BARS; i++)
            mbar_init(&bars[i], (i == P_READY || i == S_FREE || i == Q_READY) ? 8 : (i >= V_FULL0 && i <= V_FULL2) ? 4 : 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == W_MMA) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t t_o = tmem + COL_O, t_q = tmem + COL_Q, t_p = tmem + COL_P, t_s = tmem + COL_S;

    // first code row of step j (128 keys never cross a page)
    auto step_row = [&](const Kv8Layer &L, int j) -> int32_t {
        if (!L.table) return kvh * L.max_ctx + (j0 + j) * BN;
        const int id = __ldg(L.table + (size_t)kvh * L.pt_stride + (j0 + j));
        if (id < 0) report(p.status, QW_ST_BAD_PAGE);
        return max(id, 0) * QW_KV8_PAGE_TOKENS;
    };

    // Registers follow the work (per warpgroup; 2 x 168 + 64 + 112 = 4 x 128, what the block was launched with).
    if (warp >= 8 && warp < W_CV) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == W_K) {
            if (lane == 0) {
                mbar_expect_tx(&bars[Q_FULL], 4 * p.box_bytes);
                for (int b = 0; b < 4; b++) tma_load_3d(smem + OFF_STAGE_Q + b * IO_BOX, &p.qmap, b * 64, kvh * p.gqa, r0, &bars[Q_FULL]);
                for (int j = 0; j < n_t; j++) {
                    const int st = j & 1;
                    const int32_t r = step_row(p.kc, j);
                    if (j >= 2) mbar_wait(&bars[K_FREE0 + st], ((j >> 1) - 1) & 1, abort_flag, p.status, QW_ST_SLOT_TIMEOUT);
                    mbar_expect_tx(&bars[K_FULL0 + st], K_BYTES);
                    uint8_t *dst = smem + OFF_K + st * K_BYTES;
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        tma_load_2d(dst + b * KBOX, &p.kmap, b * 128, r, &bars[K_FULL0 + st]);
                        tma_load_2d(dst + b * KBOX + KBOX / 2, &p.kmap, b * 128, r + 64, &bars[K_FULL0 + st]);
                    }
                    // (the gate is wanted at the very end, with nothing left to hide a trip to memory)
                    if (j == 0 && gated)
                        for (int b = 0; b < 4; b++) prefetch_3d(&p.gmap, b * 64, kvh * p.gqa, r0);
                }
                if (gated) {
                    // the gate tile, into the K stages: both are idle once the last Q K^T has completed
                    mbar_wait(&bars[K_FREE0 + ((n_t - 1) & 1)], ((n_t - 1) >> 1) & 1, abort_flag, p.status, QW_ST_SLOT_TIMEOUT);
                    mbar_expect_tx(&bars[G_FULL], 4 * p.box_bytes);
                    for (int b = 0; b < 4; b++) tma_load_3d(smem + OFF_STAGE_IO + b * IO_BOX, &p.gmap, b * 64, kvh * p.gqa, r0, &bars[G_FULL]);
                }
            }
        } else if (warp == W_MMA) {
            if (lane == 0) {
                constexpr uint32_t idesc_qk = instr_desc(128, BN, 0);
                constexpr uint32_t hi = desc_hi(1024);
                const uint32_t k_a = smem_u32(smem + OFF_K);
                const uint32_t ql = desc_lo(smem_u32(smem + OFF_QLO), 16);
                mbar_wait(&bars[Q_READY], 0, abort_flag, p.status, QW_ST_MMA_TIMEOUT);
                for (int j = 0; j < n_t; j++) {
                    const int st = j & 1;
                    mbar_wait_hot(&bars[K_FULL0 + st], (j >> 1) & 1, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
                    if (j > 0) mbar_wait_hot(&bars[S_FREE], (j - 1) & 1, abort_flag, p.status, QW_ST_MMA_TIMEOUT);
                    // P V of step j-2 goes into the tensor queue first (the softmax threads wait for its end).  One
                    // barrier for the even and one for the odd steps: where the K tile of this step came late, P V of
                    // step j-1 has been queued too, and one barrier would be a phase ahead of the parity asked for.
                    if (j > 1) mbar_wait_hot(&bars[PV_ISSUED0 + (j & 1)], ((j >> 1) - 1) & 1, abort_flag, p.status, QW_ST_MMA_TIMEOUT);
                    tc_fence_after();
                    const uint32_t k_lo = desc_lo(k_a + st * K_BYTES, 16);
                    // 32 dims a product: 8 columns of Q high, 32 bytes inside the swizzle atom of Q low and K
#pragma unroll
                    for (int ks = 0; ks < 8; ks++) {
                        const uint32_t kd = k_lo + (ks >> 2) * (KBOX >> 4) + (ks & 3) * 2;
                        mma_ts_f8(ks > 0, t_s, t_q + ks * 8, kd, hi, idesc_qk);
                    }
#pragma unroll
                    for (int ks = 0; ks < 8; ks++) {
                        const uint32_t kd = k_lo + (ks >> 2) * (KBOX >> 4) + (ks & 3) * 2;
                        mma_ss_f8(true, t_s, ql + (ks >> 2) * (IO_BOX >> 4) + (ks & 3) * 2, hi, kd, hi, idesc_qk);
                    }
                    tc_commit(&bars[S_READY]);
                    tc_commit(&bars[K_FREE0 + st]);
                }
            }
        } else if (warp == W_PV) {
            if (lane == 0) {
                constexpr uint32_t idesc_pv = instr_desc(128, 256, 1);
                constexpr uint32_t hi = desc_hi(1024);
                const uint32_t v_a = smem_u32(smem + OFF_V);
                int st = 0;
                uint32_t ph = 0;                                 // stage and parity of the next 64 keys
                for (int j = 0; j < n_t; j++) {
                    mbar_wait_hot(&bars[V_FULL0 + st], ph, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
                    mbar_wait_hot(&bars[P_READY], j & 1, abort_flag, p.status, QW_ST_MMA_TIMEOUT);
                    tc_fence_after();
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (h == 1) {
                            mbar_wait_hot(&bars[V_FULL0 + st], ph, abort_flag, p.status, QW_ST_TMA_TIMEOUT);
                            tc_fence_after();
                        }
                        const uint32_t v_lo = desc_lo(v_a + st * V_BYTES, VBOX);
#pragma unroll
                        for (int ks = 0; ks < 4; ks++)       // 16 keys: 8 columns of P, 2048 bytes of V
                            mma_ts_f16(j > 0 || h > 0 || ks > 0, t_o, t_p + (h * 4 + ks) * 8, v_lo + ks * 128, hi, idesc_pv);
                        tc_commit(&bars[V_FREE0 + st]);
                        if (++st == V_ST) { st = 0; ph ^= 1; }
                    }
                    tc_commit(&bars[PV_DONE]);
                    mbar_arrive(&bars[PV_ISSUED0 + (j & 1)]);
                }
            }
        }
    } else if (warp >= W_CV) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        // ---------------- V codes -> fp16 ----------------
        // Eight lanes take the eight 16-byte pieces (16 dims) of half a code row, which become two 16-byte pieces of the
        // fp16 row each; lanes 4-7 of the eight write their second piece first, so that a store meets all banks.  The
        // codes of the 64 keys after the next are on their way while a stage is filled.
        const int u0 = (warp - W_CV) * 32 + lane, c = u0 & 7, k0 = u0 >> 3;
        const int n_pg = 2 * n_t;
        auto fetch = [&](uint4(&q)[8], int pg) {
            if (pg >= n_pg) return;
            const uint8_t *src = p.vc.base + ((int64_t)step_row(p.vc, pg >> 1) + (pg & 1) * 64 + k0) * 256 + c * 16;
            const int left = n_keys - (j0 * BN + pg * 64) - k0;    // keys from here on are past the last one
#pragma unroll
            for (int i = 0; i < 8; i++) {                          // half i & 1 of key k0 + 16 (i / 2)
                q[i] = make_uint4(0, 0, 0, 0);
                if (16 * (i >> 1) < left) q[i] = __ldcg(reinterpret_cast<const uint4 *>(src + (i >> 1) * 4096 + (i & 1) * 128));
            }
        };
        int st = 0;
        uint32_t ph = 1;                                           // parity of the stage's last release (first round: none)
        auto put = [&](const uint4(&q)[8], int pg) {
            if (pg >= n_pg) return;
            if (pg >= V_ST) mbar_wait(&bars[V_FREE0 + st], ph, abort_flag, p.status, QW_ST_SLOT_TIMEOUT);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int x = i & 1, key = k0 + 16 * (i >> 1);
                const uint4 a = make_uint4(f16x2_of(q[i].x), f16x2_of(q[i].x >> 16), f16x2_of(q[i].y), f16x2_of(q[i].y >> 16));
                const uint4 b = make_uint4(f16x2_of(q[i].z), f16x2_of(q[i].z >> 16), f16x2_of(q[i].w), f16x2_of(q[i].w >> 16));
                uint8_t *box = smem + OFF_V + st * V_BYTES + (x * 2 + (c >> 2)) * VBOX + key * 128;
                const uint32_t d0 = (uint32_t)(((c & 3) * 2) ^ (key & 7)) << 4, d1 = d0 ^ 16;
                const bool sw = c >= 4;
                *reinterpret_cast<uint4 *>(box + (sw ? d1 : d0)) = sw ? b : a;
                *reinterpret_cast<uint4 *>(box + (sw ? d0 : d1)) = sw ? a : b;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[V_FULL0 + st]);
            if (++st == V_ST) { st = 0; ph ^= 1; }
        };
        uint4 qa[8], qb[8];
        fetch(qa, 0);
        fetch(qb, 1);
        mbar_wait(&bars[Q_READY], 0, abort_flag, p.status, QW_ST_MMA_TIMEOUT);     // the Q tile was staged here
        for (int pg = 0; pg < n_pg; pg += 2) {
            put(qa, pg);
            fetch(qa, pg + 2);
            put(qb, pg + 1);
            fetch(qb, pg + 3);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        // ---------------- softmax + epilogue ----------------
        const int wg = warp >> 2;
        const int row_l = (warp & 3) * 32 + lane;
        const int row_r = row_l / p.gqa;
        const bool in_tile = row_r < p.tile_rows;                       // the last 128 % grouping tile rows hold nothing
        const int limit = in_tile && r0 + row_r < p.rows ? p.base_pos + r0 + row_r : n_keys - 1;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        float *xch = reinterpret_cast<float *>(smem + OFF_XCH);         // [2][2][BM]
        const uint32_t sw = row_l & 7;
        const float sc_row = stage_q(p, smem, bars, abort_flag, xch, t_q, wg, row_l, in_tile, lane_base, lane);
        uint32_t v[32];
        float m = NEG_BIG, l = 0.0f;
        const uint32_t p_cols = t_p + lane_base + wg * 32;
        const uint8_t *ke = p.kc.exps + (size_t)kvh * p.kc.exp_stride, *ve = p.vc.exps + (size_t)kvh * p.vc.exp_stride;
        const int last_blk = p.kc.exp_stride - 1;
        int ek_n = ke[min(2 * j0 + wg, last_blk)], ev_n = ve[min(2 * j0 + wg, last_blk)];
        for (int j = 0; j < n_t; j++) {
            const int ek = clamp_exp(ek_n), ev = clamp_exp(ev_n);
            if (j + 1 < n_t) {
                const int b = min(2 * (j0 + j + 1) + wg, last_blk);
                ek_n = ke[b]; ev_n = ve[b];
            }
            const float sc = fmaxf(sc_row * pow2f(ek), 1.0e-37f), fv = (float)ev;
            mbar_wait_hot(&bars[S_READY], j & 1, abort_flag, p.status, QW_ST_MMA_TIMEOUT);
            tc_fence_after();
            const int key0 = (j0 + j) * BN + wg * 64;
            uint32_t s0[32], s1[32];
            tmem_ld32(t_s + lane_base + wg * 64, s0);
            tmem_ld32(t_s + lane_base + wg * 64 + 32, s1);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[S_FREE]);
            if (key0 + 63 > p.base_pos + r0) {
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    if (key0 + e > limit) s0[e] = 0xff800000u;         // -infinity
                    if (key0 + 32 + e > limit) s1[e] = 0xff800000u;
                }
            }
            float mxa = -INFINITY, mxb = -INFINITY;
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                mxa = fmaxf(mxa, fmaxf(__uint_as_float(s0[e]), __uint_as_float(s1[e])));
                mxb = fmaxf(mxb, fmaxf(__uint_as_float(s0[e + 1]), __uint_as_float(s1[e + 1])));
            }
            // the other half's maximum (slots alternate between steps)
            float *slot = xch + (j & 1) * 2 * BM;
            const float mine = fmaf(fmaxf(mxa, mxb), sc, fv);
            slot[wg * BM + row_l] = mine;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float mx2 = fmaxf(fmaxf(mine, slot[(wg ^ 1) * BM + row_l]), NEG_BIG);
            const bool grow = j > 0 && mx2 - m > RESCALE_AT;
            const float alpha = grow ? ex2(m - mx2) : 1.0f;
            if (j == 0 || grow) m = mx2;
            const float off = fv - m + P_SHIFT;
            float la = 0.0f, lb = 0.0f;
            auto weights = [&](uint32_t(&s)[32], float &acc) {
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float x0 = ex2(fmaf(__uint_as_float(s[e]), sc, off));
                    const float x1 = ex2(fmaf(__uint_as_float(s[e + 1]), sc, off));
                    acc += x0 + x1;
                    s[e >> 1] = pack_f16(x0, x1);       // slot e/2 <= e: already consumed
                }
            };
            auto store_p = [&](const uint32_t(&s)[32], int col0) {
                uint32_t pk[16];
#pragma unroll
                for (int c = 0; c < 16; c++) pk[c] = s[c];
                tmem_st16(p_cols + col0, pk);
            };
            weights(s0, la);
            weights(s1, lb);
            l = fmaf(la + lb, pow2f(-ev), l * alpha);
            if (j > 0) {
                mbar_wait_hot(&bars[PV_DONE], (j - 1) & 1, abort_flag, p.status, QW_ST_MMA_TIMEOUT);
                tc_fence_after();
            }
            if (__any_sync(0xffffffffu, grow)) {               // both halves of a row see the same flag
#pragma unroll 1
                for (int c = 4 * wg; c < 4 * wg + 4; c++) {
                    tmem_ld32(t_o + lane_base + c * 32, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
                    tmem_st32(t_o + lane_base + c * 32, v);
                }
            }
            store_p(s0, 0);
            store_p(s1, 16);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[P_READY]);
        }
        {
            float *slot = xch + (n_t & 1) * 2 * BM;
            slot[wg * BM + row_l] = l;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            l += slot[(wg ^ 1) * BM + row_l];
        }
        mbar_wait_hot(&bars[PV_DONE], (n_t - 1) & 1, abort_flag, p.status, QW_ST_MMA_TIMEOUT);
        tc_fence_after();
        const bool elected = (warp & 3) == 0 && lane == 0;
        uint8_t *io_row = smem + OFF_STAGE_IO + row_l * 128;
        if (!whole) {
            // a share's sums: boxes of 32 dims x 128 rows as they lie in shared memory, (m, l) beside them
            if (wg == 0) stat[row_l] = make_float2(m, l);
            uint8_t *dst = reinterpret_cast<uint8_t *>(p.pacc) + (size_t)item * (8 * IO_BOX);
            const uint32_t used = (uint32_t)(min(p.tile_rows, p.rows - r0) * p.gqa) * 128;      // (tile rows past the call's end: not written)
#pragma unroll 1
            for (int c = 4 * wg; c < 4 * wg + 4; c++) {
                tmem_ld32(t_o + lane_base + c * 32, v);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 8; k++)
                    *reinterpret_cast<uint4 *>(io_row + c * IO_BOX + ((k ^ sw) << 4)) = make_uint4(v[k * 4], v[k * 4 + 1], v[k * 4 + 2], v[k * 4 + 3]);
                half_sync(wg);
                if (elected) { bulk_store(dst + c * IO_BOX, smem + OFF_STAGE_IO + c * IO_BOX, used); tma_store_commit(); }
            }
        } else {
            finish_tile(p, smem, bars, abort_flag, t_o, wg, row_l, lane_base, elected, gated, l, kvh, r0);
        }
        if (elected) tma_store_wait_read();                   // shared memory must outlive the copies
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {                                    // a wait gave up: copies and products of this CTA may still be under way
        for (int i = 0; i < 4096; i++) __nanosleep(10000);
        __syncthreads();
    }
    if (warp == W_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Adds up the shares of a tile.  A block takes 4 / SL rows of the output (a row: one head of one row of the call), SL
// slices of 64 threads x four dims each, every SL-th share, eight loads in flight.
template <int SL>
__global__ void __launch_bounds__(256) kv8_prefill_merge_kernel(const __grid_constant__ Kv8PrefillParams p) {
    __shared__ __align__(16) float acc_s[4][256];
    pdl_wait();
    pdl_launch_next();
    const int slice4 = threadIdx.x >> 6, d4 = (threadIdx.x & 63) * 4;
    const int64_t rh = (int64_t)blockIdx.x * (4 / SL) + slice4 / SL;
    const int slice = slice4 % SL;
    const bool live = rh < (int64_t)p.rows * p.q_heads;
    const int r = live ? (int)(rh / p.q_heads) : 0, h = live ? (int)(rh - (int64_t)r * p.q_heads) : 0;
    const int kvh = h / p.gqa, qt = r / p.tile_rows, i = (r - qt * p.tile_rows) * p.gqa + (h - kvh * p.gqa);
    const int item0 = ((p.n_q_tiles - 1 - qt) * p.kv_heads + kvh) * p.splits;
    const float2 *stat = reinterpret_cast<const float2 *>(p.pstat) + (size_t)item0 * BM + i;
    // dims d4 .. d4 + 3: 16-byte piece (d4 / 4) % 8 of row i in box d4 / 32
    const uint8_t *base = reinterpret_cast<const uint8_t *>(p.pacc) + (size_t)item0 * (8 * IO_BOX) + (d4 >> 5) * IO_BOX + i * 128 + ((((d4 >> 2) & 7) ^ (i & 7)) << 4);
    float m = NEG_BIG;
    for (int q = 0; q < p.splits; q++) {
        const float2 st = stat[(size_t)q * BM];
        if (st.y > 0.0f || st.y != st.y) m = fmaxf(m, st.x);
    }
    float den = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q0 = slice; q0 < p.splits; q0 += 8 * SL) {
        float4 a[8];
        float2 st[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int q = q0 + u * SL;
            st[u] = q < p.splits ? stat[(size_t)q * BM] : make_float2(NEG_BIG, 0.0f);
            a[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (q < p.splits) a[u] = *reinterpret_cast<const float4 *>(base + (size_t)q * (8 * IO_BOX));
        }
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (st[u].y == 0.0f) continue;                   // an empty share: its sums were never written
            const float f = ex2(st[u].x - m);
            den = fmaf(st[u].y, f, den);
            acc.x = fmaf(a[u].x, f, acc.x); acc.y = fmaf(a[u].y, f, acc.y); acc.z = fmaf(a[u].z, f, acc.z); acc.w = fmaf(a[u].w, f, acc.w);
        }
    }
    if (SL > 1) {
        // (the denominator: every slice has its shares' part)
        __shared__ float den_s[4];
        if ((threadIdx.x & 63) == 0) den_s[slice4] = den;
        *reinterpret_cast<float4 *>(&acc_s[slice4][d4]) = acc;
        __syncthreads();
        if (slice > 0) return;
#pragma unroll
        for (int s = 1; s < SL; s++) {
            const float4 b = *reinterpret_cast<const float4 *>(&acc_s[slice4 + s][d4]);
            acc.x += b.x; acc.y += b.y; acc.z += b.z; acc.w += b.w;
            den += den_s[slice4 + s];
        }
    }
    if (!live) return;
    const float inv = 1.0f / den;
    float o[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    if (p.gate) {
        const uint2 g = *reinterpret_cast<const uint2 *>(p.gate + (size_t)rh * p.gate_stride + d4);
        gate2(o[0], o[1], __uint_as_float(g.x << 16), __uint_as_float(g.x & 0xffff0000u));
        gate2(o[2], o[3], __uint_as_float(g.y << 16), __uint_as_float(g.y & 0xffff0000u));
    }
    *reinterpret_cast<uint2 *>(p.out + (size_t)rh * 256 + d4) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
}

}  // namespace

// How the keys of every tile are cut, and about how long the launch takes.  A step of 128 keys takes about 1.6 us, what a CTA
// does outside its steps about 9.5 us; CTAs run one per SM, so the launch takes the number of rounds times the length of a
// share, and a cut launch writes and reads up to 128 KB of sums per share on top.
// (4 kv heads: 48 query rows behind 4096 keys 15.0 us, the rule says 15.2; 499 tokens of 24 heads behind 16 K 176 and 169.)
int kv8_prefill_splits(int tiles, int steps, int sms, double *us) {
    int best = 1;
    double best_us = 0.0;
    for (int s = 1; s <= std::min(steps, 64); s++) {
        const int64_t ctas = (int64_t)tiles * s;
        if (s > 1 && ctas > 4 * sms) break;
        const double rounds = (double)((ctas + sms - 1) / sms);
        const double t = rounds * (1.6 * ((steps + s - 1) / s) + 9.5) + (s > 1 ? 0.5 + ctas * 0.03 : 0.0);
        if (s == 1 || t < best_us) { best = s; best_us = t; }
    }
    if (us) *us = best_us;
    return best;
}
size_t kv8_prefill_scratch_bytes(const Kv8PrefillParams &p) {
    return p.splits == 1 ? 0 : (size_t)p.n_q_tiles * p.kv_heads * p.splits * (8 * IO_BOX + BM * 8);
}

void launch_kv8_prefill(cudaStream_t s, Kv8PrefillParams &p, void *scratch) {
    static bool configured[64] = {false};      // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        cudaFuncSetAttribute(kv8_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
        configured[dev] = true;
    }
    const size_t items = (size_t)p.n_q_tiles * p.kv_heads * p.splits;
    p.pacc = reinterpret_cast<float *>(scratch);
    p.pstat = p.splits == 1 ? nullptr : p.pacc + items * (8 * IO_BOX / 4);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = cudaLaunchConfig_t();
    cfg.gridDim = dim3((unsigned)items); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM_BYTES; cfg.stream = s;
    cfg.attrs = &attr; cfg.numAttrs = g_tune_pdl ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kv8_prefill_kernel, p);
    g_launches++;
    if (p.splits == 1) return;
    const int64_t rh = (int64_t)p.rows * p.q_heads;
    const bool wide = p.splits > 4;
    cfg.gridDim = dim3((unsigned)(wide ? rh : (rh + 3) / 4)); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = 0;
    if (wide) cudaLaunchKernelEx(&cfg, kv8_prefill_merge_kernel<4>, p);
    else cudaLaunchKernelEx(&cfg, kv8_prefill_merge_kernel<1>, p);
    g_launches++;
}

}  // namespace qw
