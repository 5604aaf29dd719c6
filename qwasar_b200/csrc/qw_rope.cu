// Rotary positions in both layouts (sm_100a).
//
// Pair j of a head turns by a = pos * inv_freq[j]:
//     (x1, x2) -> amp * (x1 cos a - x2 sin a,  x2 cos a + x1 sin a)
// with the pair's two elements half a rotated part apart (half layout) or side by side (interleaved).
//
// The angle reaches 10^6 radians, where a 32-bit product is off by hundredths of a radian: it is formed
// and reduced modulo 2 pi in 64 bits (error below 1e-9), and only the remainder goes to the 32-bit sine
// and cosine.  Those cost more than the rotation itself, so a block works out the angles of one row once,
// in shared memory, and uses them for all the heads it takes.
//
// Memory bounds it: 4096 rows of 24 heads x 256, bf16, interleaved, 18.0 us, of which the bytes take 15.4 (blocks of 256
// threads with fewer vectors on their way: 20.8).  One row of 16 heads: 1.6 us, the launch.
#include "qw_kernels.h"

namespace qw {

namespace {

constexpr int ROPE_THREADS = 128, FLY = 3;        // vectors (half layout: pairs of vectors) a thread has on their way at a time
constexpr int ROPE_ITEMS = FLY * ROPE_THREADS;    // what a block takes at once: beyond that the heads are split over more blocks

template <typename T> struct Vec;                 // 16 bytes of T
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(float (&v)[4], uint4 t) {
        v[0] = __uint_as_float(t.x); v[1] = __uint_as_float(t.y); v[2] = __uint_as_float(t.z); v[3] = __uint_as_float(t.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(float (&v)[8], uint4 t) {
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
};
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float *p, float v) { *p = v; }
__device__ __forceinline__ void from_f(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// One block: one row, heads [head0, head0 + n).  VEC: every access is a whole aligned 16-byte vector.
template <typename T, bool VEC, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeParams p, int heads_per_block) {
    extern __shared__ float2 cs[];                // (cos, sin) * amp of the row's rotary_dim / 2 angles
    pdl_wait();
    pdl_launch_next();
    const int row = blockIdx.x, half = p.rotary_dim >> 1;
    const int head0 = blockIdx.y * heads_per_block, nh = min(heads_per_block, p.heads - head0);
    const T *x = reinterpret_cast<const T *>(p.x) + (size_t)row * p.x_stride + (size_t)head0 * p.head_dim;
    T *y = reinterpret_cast<T *>(p.y) + (size_t)row * p.y_stride + (size_t)head0 * p.head_dim;
    const bool copy = (const void *)p.x != (const void *)p.y;     // in place: the dims that do not turn stay where they are
    constexpr int N = VEC ? Vec<T>::N : 1;
    // items of one head: rotations (N pairs each in the half layout, N / 2 or 1 in the interleaved one), then copies
    const int per_rot = (INTER && VEC) ? N / 2 : N;
    const int n_rot = half / per_rot, n_cp = copy ? (p.head_dim - p.rotary_dim) / N : 0;
    const int per = n_rot + n_cp, total = nh * per;
    // (the first vectors are asked for in front of the angles)
    uint4 a[FLY], b[FLY];
    int off[FLY], idx[FLY];
    auto fetch = [&](int it0) {
#pragma unroll
        for (int f = 0; f < FLY; f++) {
            const int it = it0 + f * ROPE_THREADS;
            const int h = it / per, i = it - h * per;
            idx[f] = it < total ? i : -1;
            off[f] = h * p.head_dim + (i < n_rot ? i * N : p.rotary_dim + (i - n_rot) * N);
            if (it < total) {
                a[f] = *reinterpret_cast<const uint4 *>(x + off[f]);
                if (!INTER && i < n_rot) b[f] = *reinterpret_cast<const uint4 *>(x + off[f] + half);
            }
        }
    };
    if constexpr (VEC) fetch(threadIdx.x);
    const double pos = (double)p.pos[row];
    for (int j = threadIdx.x; j < half; j += ROPE_THREADS) {
        const double a = pos * (double)p.inv_freq[j];
        const double turns = rint(a * 0.15915494309189533577);
        // 2 pi in two parts: the product turns * 2pi_hi is exact in the fused operation
        const float r = (float)fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586477, a));
        float s, c;
        sincosf(r, &s, &c);
        cs[j] = make_float2(c * p.amp, s * p.amp);
    }
    __syncthreads();
    if constexpr (VEC) {
        for (int it0 = threadIdx.x; it0 < total; it0 += FLY * ROPE_THREADS) {
            if (it0 != (int)threadIdx.x) fetch(it0);
#pragma unroll
            for (int f = 0; f < FLY; f++) {
                if (idx[f] < 0) break;
                T *o = y + off[f];
                if (idx[f] >= n_rot) { *reinterpret_cast<uint4 *>(o) = a[f]; continue; }
                float u[N];
                Vec<T>::unpack(u, a[f]);
                if constexpr (INTER) {
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        const float2 t = cs[idx[f] * (N / 2) + e / 2];
                        const float p0 = u[e], p1 = u[e + 1];
                        u[e] = p0 * t.x - p1 * t.y;
                        u[e + 1] = p1 * t.x + p0 * t.y;
                    }
                } else {
                    float v[N];
                    Vec<T>::unpack(v, b[f]);
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const float2 t = cs[idx[f] * N + e];
                        const float p0 = u[e], p1 = v[e];
                        u[e] = p0 * t.x - p1 * t.y;
                        v[e] = p1 * t.x + p0 * t.y;
                    }
                    *reinterpret_cast<uint4 *>(o + half) = Vec<T>::pack(v);
                }
                *reinterpret_cast<uint4 *>(o) = Vec<T>::pack(u);
            }
        }
    } else {
        for (int it = threadIdx.x; it < total; it += ROPE_THREADS) {
            const int h = it / per, i = it - h * per;
            const T *xh = x + (size_t)h * p.head_dim;
            T *yh = y + (size_t)h * p.head_dim;
            if (i >= n_rot) {
                const int d = p.rotary_dim + i - n_rot;
                yh[d] = xh[d];
            } else {
                const int d0 = INTER ? 2 * i : i, d1 = INTER ? 2 * i + 1 : i + half;
                const float2 t = cs[i];
                const float u = to_f(xh[d0]), v = to_f(xh[d1]);
                from_f(yh + d0, u * t.x - v * t.y);
                from_f(yh + d1, v * t.x + u * t.y);
            }
        }
    }
}

template <typename T, bool VEC, bool INTER>
void launch_t(cudaStream_t s, const RopeParams &p) {
    constexpr int N = VEC ? Vec<T>::N : 1;
    const int items = (p.rotary_dim / 2) / ((INTER && VEC) ? N / 2 : N) + (p.head_dim - p.rotary_dim) / N;
    int hpb = ROPE_ITEMS / (items > 0 ? items : 1);
    if (hpb < 1) hpb = 1;
    if (hpb > p.heads) hpb = p.heads;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = cudaLaunchConfig_t();
    cfg.gridDim = dim3((unsigned)p.rows, (unsigned)((p.heads + hpb - 1) / hpb)); cfg.blockDim = dim3(ROPE_THREADS);
    cfg.dynamicSmemBytes = (size_t)(p.rotary_dim / 2) * sizeof(float2); cfg.stream = s;
    cfg.attrs = &attr; cfg.numAttrs = g_tune_pdl ? 1 : 0;
    cudaLaunchKernelEx(&cfg, rope_kernel<T, VEC, INTER>, p, hpb);
    g_launches++;
}

template <typename T>
void launch_io(cudaStream_t s, const RopeParams &p) {
    constexpr int N = Vec<T>::N;
    // whole vectors: rows, heads and the two halves of the rotated part all start on 16 bytes
    const int half = p.rotary_dim / 2;
    const bool vec = p.x_stride % N == 0 && p.y_stride % N == 0 && p.head_dim % N == 0 && p.rotary_dim % N == 0 &&
                     (p.interleaved || half % N == 0);
    if (vec) { if (p.interleaved) launch_t<T, true, true>(s, p); else launch_t<T, true, false>(s, p); }
    else { if (p.interleaved) launch_t<T, false, true>(s, p); else launch_t<T, false, false>(s, p); }
}

}  // namespace

void launch_rope(cudaStream_t s, const RopeParams &p) {
    if (p.io == DT_BF16) launch_io<__nv_bfloat16>(s, p);
    else launch_io<float>(s, p);
}

}  // namespace qw
