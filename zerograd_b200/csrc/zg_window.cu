// zg_window.cu -- causal attention over long sequences, with a sliding window
// and a few first tokens that stay visible (sinks):
//
//   o[z, i, h] = sum_j softmax_j(q[z, i, h] . k[z, j, h / G] / sqrt(D)) v[z, j, h / G]
//   over j <= i with i - j < window or j < sinks, i, j < length[z]
//
// q, o [Z, S, H, D], k, v [Z, S, K, D], G = H / K.  Rows i >= length[z] are
// zeros.  4 D flops for each visible (i, j) and head.
#include <math.h>

#include "zg_ptx.cuh"
#include "zg_tc.cuh"

namespace {

struct WindowArgs {
    const void *q, *k, *v;
    void* o;
    const int32_t* lengths;
    int64_t ldq, ldk, ldv;
    int Z, S, H, K, D, G;
    int window, sinks;  // window >= 1 (S where there is none)
    float scale;        // log2(e) / sqrt(D)
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The length of sequence z; -1 when it is not one of [0, S].
__device__ __forceinline__ int length_of(const WindowArgs& a, int z) {
    if (!a.lengths) return a.S;
    const int n = a.lengths[z];
    return n < 0 || n > a.S ? -1 : n;
}

// Whether position i sees position j <= i.
__device__ __forceinline__ bool sees(const WindowArgs& a, int i, int j) { return i - j < a.window || j < a.sinks; }

// One output row by one warp, each visible key on its own in float32: what
// the tiled kernels fall back to for a row that came out not finite.  A key
// or value of a masked place that is infinite or NaN has a weight of zero,
// and a tile's product would turn 0 * inf into NaN; here it is not read.
template <typename T>
__device__ __noinline__ void window_row(const WindowArgs& a, int z, int i, int h) {
    const int lane = threadIdx.x % 32;
    const int kh = h / a.G;
    const T* q = static_cast<const T*>(a.q) + ((int64_t)z * a.S + i) * a.ldq + (int64_t)h * a.D;
    const T* k = static_cast<const T*>(a.k) + (int64_t)z * a.S * a.ldk + (int64_t)kh * a.D;
    const T* v = static_cast<const T*>(a.v) + (int64_t)z * a.S * a.ldv + (int64_t)kh * a.D;
    T* o = static_cast<T*>(a.o) + (((int64_t)z * a.S + i) * a.H + h) * a.D;
    float qv[8], x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = lane + 32 * e;
        qv[e] = d < a.D ? zg_to_float(q[d]) * a.scale : 0.f;
        x[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j <= i; ++j) {
        if (!sees(a, i, j)) {
            j = i - a.window;  // the window's first position is next
            continue;
        }
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = lane + 32 * e;
            if (d < a.D) s = fmaf(qv[e], zg_to_float(k[j * a.ldk + d]), s);
        }
#pragma unroll
        for (int f = 16; f > 0; f >>= 1) s += __shfl_xor_sync(0xffffffffu, s, f);
        const float n = fmaxf(m, s), base = n == -INFINITY ? 0.f : n;
        const float c = exp2f(m - base), p = exp2f(s - base);
        l = fmaf(l, c, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = lane + 32 * e;
            if (d < a.D) x[e] = fmaf(p, zg_to_float(v[j * a.ldv + d]), x[e] * c);
        }
        m = n;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = lane + 32 * e;
        if (d < a.D) o[d] = zg_from_float<T>(x[e] / l);
    }
}

// ---------------------------------------------------------------------------
// FMA path: float32, and bf16 shapes that the tensor cores do not take.
//
// A block has 64 query rows of one head and walks over the tiles of 64 keys
// that any of them sees, q, k, v and the weights in shared memory as float32.
// 256 threads as 16 x 16: thread (ty, tx) has the scores of rows ty + 16 i
// and keys tx + 16 j, and the outputs of the same rows in columns
// 4 tx + 64 c.  Rows are DP + 4 floats apart, so that the 16-byte reads of
// neighbouring rows fall into different banks.
// ---------------------------------------------------------------------------
constexpr int WF_M = 64, WF_N = 64, WF_THREADS = 256, WF_PP = WF_N + 4;

template <int DP>
constexpr size_t wf_smem() {
    return (size_t)(3 * 64 * (DP + 4) + WF_M * WF_PP) * sizeof(float);
}

template <typename T, int DP>
__global__ void __launch_bounds__(WF_THREADS) window_fma_kernel(const WindowArgs a, int q_tiles, int vec) {
    constexpr int PITCH = DP + 4, NC = DP / 64;
    extern __shared__ __align__(16) float sm[];
    float *qs = sm, *ks = qs + 64 * PITCH, *vs = ks + 64 * PITCH, *ps = vs + 64 * PITCH;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    // the tiles that see the most keys first
    const int qt = q_tiles - 1 - (int)(blockIdx.x % q_tiles);
    const int64_t zh = blockIdx.x / q_tiles;
    const int z = (int)(zh / a.H), h = (int)(zh % a.H), kh = h / a.G;
    const int n = length_of(a, z), i0 = qt * WF_M;
    T* o = static_cast<T*>(a.o) + ((int64_t)z * a.S * a.H + h) * a.D;
    const int64_t ldo = (int64_t)a.H * a.D;
    if (i0 >= n) {  // rows behind the sequence
        for (int x = threadIdx.x; x < WF_M * a.D; x += WF_THREADS) {
            const int i = i0 + x / a.D;
            if (i < a.S) o[i * ldo + x % a.D] = zg_from_float<T>(n < 0 ? __int_as_float(0x7fffffff) : 0.f);
        }
        return;
    }
    const T* q = static_cast<const T*>(a.q) + (int64_t)z * a.S * a.ldq + (int64_t)h * a.D;
    const T* k = static_cast<const T*>(a.k) + (int64_t)z * a.S * a.ldk + (int64_t)kh * a.D;
    const T* v = static_cast<const T*>(a.v) + (int64_t)z * a.S * a.ldv + (int64_t)kh * a.D;

    auto load = [&](float* dst, const T* src, int64_t ld, int r0) {  // 64 rows from r0, zeros past n and D
        if (vec) {
            for (int x = threadIdx.x; x < 64 * (DP / 4); x += WF_THREADS) {
                const int r = x / (DP / 4), d = x % (DP / 4) * 4;
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r0 + r < n && d < a.D) {
                    const T* p = src + (r0 + r) * ld + d;
                    if constexpr (sizeof(T) == 4) {
                        f = *reinterpret_cast<const float4*>(p);
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2*>(p);
                        f = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                                        __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
                    }
                }
                *reinterpret_cast<float4*>(dst + r * PITCH + d) = f;
            }
        } else {
            for (int x = threadIdx.x; x < 64 * DP; x += WF_THREADS) {
                const int r = x / DP, d = x % DP;
                dst[r * PITCH + d] = r0 + r < n && d < a.D ? zg_to_float(src[(r0 + r) * ld + d]) : 0.f;
            }
        }
    };
    load(qs, q, a.ldq, i0);

    float x[4][4 * NC], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4 * NC; ++c) x[i][c] = 0.f;
    }
    const int last = i0 + WF_M < n ? i0 + WF_M : n;  // rows [i0, last)
    const int kt_end = (last + WF_N - 1) / WF_N;
    const int w0 = i0 - a.window + 1 > 0 ? (i0 - a.window + 1) / WF_N : 0;  // the window's first tile
    int sink_end = (a.sinks + WF_N - 1) / WF_N;                              // tiles that hold sinks
    if (sink_end > w0) sink_end = w0;
    for (int kt = sink_end > 0 ? 0 : w0; kt < kt_end; kt = kt + 1 < sink_end || kt >= w0 ? kt + 1 : w0) {
        const int j0 = kt * WF_N;
        __syncthreads();  // the last tile has been read
        load(ks, k, a.ldk, j0);
        load(vs, v, a.ldv, j0);
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
        for (int d = 0; d < DP; d += 4) {
            float4 qv[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                qv[i] = *reinterpret_cast<const float4*>(qs + (ty + 16 * i) * PITCH + d);
                kv[i] = *reinterpret_cast<const float4*>(ks + (tx + 16 * i) * PITCH + d);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[i][j] = fmaf(qv[i].x, kv[j].x,
                                   fmaf(qv[i].y, kv[j].y, fmaf(qv[i].z, kv[j].z, fmaf(qv[i].w, kv[j].w, s[i][j]))));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int qi = i0 + ty + 16 * i;
            float t = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int kj = j0 + tx + 16 * j;
                s[i][j] = kj <= qi && kj < n && sees(a, qi, kj) ? s[i][j] * a.scale : -INFINITY;
                t = fmaxf(t, s[i][j]);
            }
#pragma unroll
            for (int f = 8; f > 0; f >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, f));
            const float base = t == -INFINITY ? 0.f : t;
            const float c = exp2f(m[i] - base);
            m[i] = t;
            l[i] *= c;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(s[i][j] - base);
                l[i] += p;
                ps[(ty + 16 * i) * WF_PP + tx + 16 * j] = p;
            }
#pragma unroll
            for (int e = 0; e < 4 * NC; ++e) x[i][e] *= c;
        }
        __syncwarp();  // a row's weights are written and read by the same half warp
#pragma unroll 2
        for (int j = 0; j < WF_N; j += 4) {
            float4 pv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = *reinterpret_cast<const float4*>(ps + (ty + 16 * i) * WF_PP + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float4 vv = *reinterpret_cast<const float4*>(vs + (j + e) * PITCH + 64 * c + 4 * tx);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = e == 0 ? pv[i].x : e == 1 ? pv[i].y : e == 2 ? pv[i].z : pv[i].w;
                        x[i][4 * c] = fmaf(p, vv.x, x[i][4 * c]);
                        x[i][4 * c + 1] = fmaf(p, vv.y, x[i][4 * c + 1]);
                        x[i][4 * c + 2] = fmaf(p, vv.z, x[i][4 * c + 2]);
                        x[i][4 * c + 3] = fmaf(p, vv.w, x[i][4 * c + 3]);
                    }
                }
            }
        }
        __syncwarp();
    }
    unsigned redo = 0;  // bit i: row i of this half warp is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int f = 8; f > 0; f >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], f);
        const int qi = i0 + ty + 16 * i;
        bool fine = true;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 64 * c + 4 * tx + e;
                const float y = qi < n ? x[i][4 * c + e] / l[i] : 0.f;
                if (d < a.D) {
                    fine = fine && isfinite(y);
                    if (qi < a.S) o[qi * ldo + d] = zg_from_float<T>(y);
                }
            }
        const unsigned half = 0xffffu << (threadIdx.x % 32 / 16 * 16);
        if (__ballot_sync(0xffffffffu, !fine) & half) redo |= 1u << i;
    }
    // the rows of this warp's two halves, one at a time by the whole warp
    for (int t = 0; t < 2; ++t) {
        const unsigned rows = __shfl_sync(0xffffffffu, redo, 16 * t);
        for (int i = 0; i < 4; ++i)
            if (rows >> i & 1) {
                __syncwarp();  // the row's first values are written before these
                window_row<T>(a, z, i0 + (int)(threadIdx.x / 32) * 2 + t + 16 * i, h);
            }
    }
}

template <typename T, int DP>
int launch_window_fma(const WindowArgs& a, int vec, cudaStream_t st) {
    const size_t smem = wf_smem<DP>();
    if (cudaFuncSetAttribute(window_fma_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
        cudaSuccess)
        return zg::fail(ZG_ERR_CUDA, "zg_window_attention: shared memory attribute");
    const int q_tiles = (a.S + WF_M - 1) / WF_M;
    const int64_t blocks = (int64_t)a.Z * a.H * q_tiles;
    if (blocks > INT32_MAX) return zg::fail(ZG_ERR_INVALID, "zg_window_attention: too many rows");
    zg::LaunchTimer zg_lt_("window_attention_fma", st);
    window_fma_kernel<T, DP><<<(unsigned)blocks, WF_THREADS, smem, st>>>(a, q_tiles, vec);
    return zg::check_launch("zg_window_attention");
}

template <typename T>
int launch_window_any(const WindowArgs& a, cudaStream_t st) {
    auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const int vec = a.D % 4 == 0 && a.ldq % 4 == 0 && a.ldk % 4 == 0 && a.ldv % 4 == 0 && al(a.q) && al(a.k) && al(a.v);
    return a.D <= 64    ? launch_window_fma<T, 64>(a, vec, st)
           : a.D <= 128 ? launch_window_fma<T, 128>(a, vec, st) : launch_window_fma<T, 256>(a, vec, st);
}

}  // namespace

extern "C" int zg_window_attention(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                   const int32_t* lengths, int64_t Z, int64_t S, int H, int K, int D, int window,
                                   int sinks, int dtype, void* o, void* stream) {
    if (Z < 0 || S < 0 || Z > INT32_MAX || S > (1 << 30) || H < 1 || K < 1 || H % K || D < 1)
        return zg::fail(ZG_ERR_INVALID, "zg_window_attention: bad sizes");
    if (D > 256) return zg::fail(ZG_ERR_UNSUPPORTED, "zg_window_attention: head dim above 256");
    if (window < 0 || sinks < 0)
        return zg::fail(ZG_ERR_INVALID, "zg_window_attention: window and sinks must be >= 0");
    if (ldq < (int64_t)H * D || ldk < (int64_t)K * D || ldv < (int64_t)K * D)
        return zg::fail(ZG_ERR_INVALID, "zg_window_attention: row pitch below heads * D");
    if (!zg::dtype_ok(dtype)) return zg::fail(ZG_ERR_INVALID, "zg_window_attention: bad dtype");
    if (Z == 0 || S == 0) return ZG_OK;
    if (!q || !k || !v || !o) return zg::fail(ZG_ERR_INVALID, "zg_window_attention: null pointer");
    const WindowArgs a{q, k, v, o, lengths, ldq, ldk, ldv, (int)Z, (int)S, H, K, D, H / K,
                       window > 0 && window < S ? window : (int)S, sinks < S ? sinks : (int)S,
                       (float)(1.4426950408889634 / sqrt((double)D))};
    cudaStream_t st = zg::as_stream(stream);
    return dtype == ZG_BF16 ? launch_window_any<__nv_bfloat16>(a, st) : launch_window_any<float>(a, st);
}
