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

// ---------------------------------------------------------------------------
// Tensor-core path: bf16, D <= DP (64 or 128, zeros behind D).
//
// A persistent CTA per SM, 384 threads: warp 0 issues the TMA loads, warp 1
// the MMAs, warps 4-7 and 8-11 are the softmax groups of two tiles of 128
// query rows (one thread a row).  A work unit is a pair of neighbouring
// tiles of one (z, head), so that each block of 128 keys and values is
// fetched once for both; the units with the most visible keys come first.
// Per block and tile: S = Q K^T into TMEM (M = N = 128), a row's maximum, the
// weights p = 2^(s - m) as bf16 back into TMEM, O += P V with P read from
// TMEM.  While one tile's group is at its weights, the tensor cores work for
// the other.  Only blocks that a tile sees any key of are visited, and only
// those at the edge of the mask test each key.
//
// The maximum m that weights are taken against is moved, and O rescaled by
// its group, only when a row's true maximum is more than 2^8 above it: the
// quotient O / l is the same, weights stay below 2^8 (and their relative
// rounding in bf16 is what it was), and after the first blocks O is hardly
// ever touched.
//
// TMEM (512 columns): S of the two tiles, O of the two tiles, and P: with
// DP = 64 in columns of its own, so the next block's Q K^T is issued before P V
// and runs under the next softmax; with DP = 128 over the scores it came from
// (no column is left), so the next Q K^T waits for P V to have read it.
// ---------------------------------------------------------------------------
constexpr int WT_THREADS = 384;
constexpr int WT_BLOCK = 128;  // keys of a block, rows of a tile

template <int DP>
struct WtShape {
    static constexpr uint32_t TILE = 128 * DP * 2;       // bytes of a tile of rows: DP / 64 boxes of 128 x 64
    static constexpr int STAGES = DP == 64 ? 8 : 5;      // ring of key and value blocks
    static constexpr uint32_t RING = 2 * TILE;           // behind the two query tiles
    static constexpr uint32_t CTRL = RING + STAGES * TILE;
    static constexpr uint32_t SMEM = CTRL + 512;
    static constexpr bool OWN_P = DP == 64;
    // TMEM columns of tile t's scores, weights and outputs
    static __device__ __forceinline__ uint32_t s_col(int t) { return t * 128; }
    static __device__ __forceinline__ uint32_t p_col(int t) { return OWN_P ? 384 + t * 64 : t * 128; }
    static __device__ __forceinline__ uint32_t o_col(int t) { return 256 + t * DP; }
};

struct WtCtrl {
    uint64_t q_full, q_empty, kv_full[8], kv_empty[8], s_full[2], p_full[2], pv_done[2], o_empty[2], done;
    uint32_t tmem_base;
};
static_assert(sizeof(WtCtrl) <= 512, "control block");

// A unit: two tiles of 128 rows from i0, the blocks of keys that they see.
struct WtUnit {
    int z, h, n, i0, sink_blocks, hi;
    int lo[2];  // the first block of the tile's window
    __device__ __forceinline__ bool alive(int t) const { return i0 + 128 * t < n; }
    __device__ __forceinline__ int diag(int t) const { return i0 / WT_BLOCK + t; }
    // whether tile t sees any key of block b
    __device__ __forceinline__ bool takes(int t, int b) const {
        return alive(t) && b <= diag(t) && (b >= lo[t] || b < sink_blocks);
    }
    __device__ __forceinline__ int first() const { return sink_blocks > 0 ? 0 : lo[0]; }
    __device__ __forceinline__ int next(int b) const { return b + 1 < sink_blocks || b + 1 >= lo[0] ? b + 1 : lo[0]; }
};

__device__ __forceinline__ WtUnit wt_unit(const WindowArgs& a, int64_t u, int pairs) {
    WtUnit x;
    const int64_t zh_count = (int64_t)a.Z * a.H;
    const int pair = pairs - 1 - (int)(u / zh_count);
    const int64_t zh = u % zh_count;
    x.z = (int)(zh / a.H);
    x.h = (int)(zh % a.H);
    x.n = length_of(a, x.z);
    x.i0 = pair * 256;
    x.sink_blocks = (a.sinks + WT_BLOCK - 1) / WT_BLOCK;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int w = x.i0 + 128 * t - a.window + 1;
        x.lo[t] = w > 0 ? w / WT_BLOCK : 0;
    }
    x.hi = x.diag(x.alive(1) ? 1 : 0);
    return x;
}

// Bits 0 .. x of a word.
__device__ __forceinline__ uint32_t bits_upto(int x) { return x < 0 ? 0u : x >= 31 ? 0xffffffffu : (2u << x) - 1u; }

// The keys jc .. jc + 31 that row i of a sequence of n sees, as bits.
__device__ __forceinline__ uint32_t seen_bits(const WindowArgs& a, int i, int n, int jc) {
    const int last = i < n - 1 ? i : n - 1;
    return bits_upto(last - jc) & (~bits_upto(i - a.window - jc) | bits_upto(a.sinks - 1 - jc));
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}

template <int DP>
__global__ void __launch_bounds__(WT_THREADS, 1)
window_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const WindowArgs a, int pairs, int64_t units) {
    using W = WtShape<DP>;
    // No static shared memory, so the dynamic block starts at the CTA's first
    // shared byte; the swizzled tiles need it 1024-aligned, which is checked.
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicCAS(&g_zg_tc_error, 0u, 109u);
        return;
    }
    WtCtrl& c = *reinterpret_cast<WtCtrl*>(smem + W::CTRL);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        mbar_init(&c.q_full, 1);
        mbar_init(&c.q_empty, 1);
        mbar_init(&c.done, 1);
        for (int i = 0; i < W::STAGES; ++i) {
            mbar_init(&c.kv_full[i], 1);
            mbar_init(&c.kv_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&c.s_full[t], 1);
            mbar_init(&c.p_full[t], 128);
            mbar_init(&c.pv_done[t], 1);
            mbar_init(&c.o_empty[t], 128);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(&c.tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = c.tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t slot = 0, nq = 0, issued = 0;  // loads issued; a stage's parity follows from the count
            bool ok = true;
            for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x) {
                const WtUnit x = wt_unit(a, u, pairs);
                if (!x.alive(0)) continue;
                const int kh = x.h / a.G, tiles = x.alive(1) ? 2 : 1;
                if (!(ok = mbar_wait(&c.q_empty, (nq & 1) ^ 1, 101))) break;
                mbar_expect_tx(&c.q_full, tiles * W::TILE);
                for (int t = 0; t < tiles; ++t)
                    for (int d = 0; d < DP / 64; ++d)
                        tma_load_4d(smem + t * W::TILE + d * 16384, &tmQ, &c.q_full, 64 * d, x.h, x.i0 + 128 * t, x.z);
                ++nq;
                for (int b = x.first(); ok && b <= x.hi; b = x.next(b))
                    for (int v = 0; v < 2; ++v, ++slot) {
                        const uint32_t st = slot % W::STAGES;
                        if (!(ok = mbar_wait(&c.kv_empty[st], ((slot / W::STAGES) & 1) ^ 1, 102))) break;
                        mbar_expect_tx(&c.kv_full[st], W::TILE);
                        for (int d = 0; d < DP / 64; ++d)
                            tma_load_4d(smem + W::RING + st * W::TILE + d * 16384, v ? &tmV : &tmK, &c.kv_full[st], 64 * d,
                                        kh, b * WT_BLOCK, x.z);
                        issued = slot + 1;
                    }
            }
            // loads still in flight (only after an abort) land before the CTA exits
            for (uint32_t s = issued > W::STAGES ? issued - W::STAGES : 0; s < issued; ++s)
                for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&c.kv_full[s % W::STAGES], (s / W::STAGES) & 1); ++i) {
                }
            if (nq)
                for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&c.q_full, (nq - 1) & 1); ++i) {
                }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc_s = idesc_bf16(128, 128, 0), idesc_o = idesc_bf16(128, DP, 1);
            uint32_t slot = 0, nq = 0, ns[2] = {0, 0}, npv[2] = {0, 0}, nu[2] = {0, 0};
            bool ok = true;
            for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x) {
                const WtUnit x = wt_unit(a, u, pairs);
                if (!x.alive(0)) continue;
                if (!(ok = mbar_wait(&c.q_full, nq & 1, 103))) break;
                ++nq;
                bool pending[2] = {false, false}, started[2] = {false, false};
                // S of tile t from the key block in slot sk
                auto scores = [&](int t, uint32_t sk) {
                    const uint32_t qa = smem_u32(smem + t * W::TILE), ka = smem_u32(smem + W::RING + sk % W::STAGES * W::TILE);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        umma_bf16(tmem + W::s_col(t), smem_desc(qa + (k / 4) * 16384 + (k % 4) * 32, 16, 1024),
                                  smem_desc(ka + (k / 4) * 16384 + (k % 4) * 32, 16, 1024), idesc_s, k > 0 ? 1u : 0u);
                    umma_commit(&c.s_full[t]);
                    ++ns[t];
                };
                // O of tile t += its weights times the value block in slot sv
                auto outputs = [&](int t, uint32_t sv) {
                    const uint32_t va = smem_u32(smem + W::RING + sv % W::STAGES * W::TILE);
#pragma unroll
                    for (int k = 0; k < WT_BLOCK / 16; ++k)
                        umma_bf16_ts(tmem + W::o_col(t), tmem + W::p_col(t) + k * 8, smem_desc(va + k * 2048, 16384, 1024),
                                     idesc_o, started[t] || k > 0 ? 1u : 0u);
                    umma_commit(&c.pv_done[t]);
                    ++npv[t];
                    started[t] = true;
                    pending[t] = false;
                };
                // one step: the weights of the last block (if a tile has any) and the scores of block b (b < 0: none)
                auto step = [&](int b, uint32_t sk) {
                    bool v_ready = false;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        bool need = b >= 0 && x.takes(t, b);
                        if (pending[t]) {
                            if (!mbar_wait(&c.p_full[t], (ns[t] - 1) & 1, 104)) return false;
                            tc_fence_after();
                            if (W::OWN_P && need) {
                                scores(t, sk);
                                need = false;
                            }
                            if (!v_ready && !mbar_wait(&c.kv_full[(sk - 1) % W::STAGES], ((sk - 1) / W::STAGES) & 1, 105))
                                return false;
                            v_ready = true;
                            if (!started[t]) {
                                // the last unit's outputs have been read
                                if (!mbar_wait(&c.o_empty[t], (nu[t] & 1) ^ 1, 106)) return false;
                                ++nu[t];
                            }
                            tc_fence_after();
                            outputs(t, sk - 1);
                            if (W::OWN_P && b >= 0 && x.takes(t, b)) pending[t] = true;
                        }
                        if (need) {
                            // P shares the scores' columns: it has been read
                            if (!W::OWN_P && npv[t] > 0 && !mbar_wait(&c.pv_done[t], (npv[t] - 1) & 1, 107)) return false;
                            scores(t, sk);
                            pending[t] = true;
                        }
                    }
                    return true;
                };
                const uint32_t s0 = slot;
                for (int b = x.first(); ok && b <= x.hi; b = x.next(b), slot += 2) {
                    if (!(ok = mbar_wait(&c.kv_full[slot % W::STAGES], (slot / W::STAGES) & 1, 108))) break;
                    tc_fence_after();
                    if (!(ok = step(b, slot))) break;
                    if (slot > s0) umma_commit(&c.kv_empty[(slot - 1) % W::STAGES]);
                    umma_commit(&c.kv_empty[slot % W::STAGES]);
                }
                if (!ok) break;
                umma_commit(&c.q_empty);
                if (!(ok = step(-1, slot))) break;
                umma_commit(&c.kv_empty[(slot - 1) % W::STAGES]);
            }
            // every MMA this thread issued has completed before TMEM is freed
            umma_commit(&c.done);
            for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&c.done, 0); ++i) {
            }
        }
    } else if (warp >= 4) {
        const int t = (warp - 4) / 4, quad = warp % 4;
        const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t sc = trow + W::s_col(t), pc = trow + W::p_col(t), oc = trow + W::o_col(t);
        const int64_t ldo = (int64_t)a.H * a.D;
        uint32_t nb = 0;  // blocks of this tile so far
        bool ok = true;
        for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x) {
            const WtUnit x = wt_unit(a, u, pairs);
            const int row0 = x.i0 + 128 * t, i = row0 + 32 * quad + lane;
            __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.o) + ((int64_t)x.z * a.S + i) * ldo + (int64_t)x.h * a.D;
            if (!x.alive(t)) {
                if (i < a.S) {
                    const uint32_t w = x.n < 0 ? 0x7fff7fffu : 0u;
                    for (int d = 0; d < a.D; d += 8) *reinterpret_cast<uint4*>(o + d) = make_uint4(w, w, w, w);
                }
                continue;
            }
            float m = -INFINITY;  // what the weights are taken against, in units of log2
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            bool first = true;
            for (int b = x.first(); b <= x.hi; b = x.next(b)) {
                if (!x.takes(t, b)) continue;
                if (!(ok = warp_wait(&c.s_full[t], nb & 1, 110))) break;
                tc_fence_after();
                const int j0 = b * WT_BLOCK;
                const bool edge = j0 + WT_BLOCK - 1 > row0 ||
                                  (j0 <= row0 + 127 - a.window && j0 + WT_BLOCK > a.sinks);
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                {
                    uint32_t r[2][32];
                    tmem_ld32_nowait(sc, r[0]);
#pragma unroll 2
                    for (int q = 0; q < 4; ++q) {
                        tmem_wait_ld32(r[q & 1]);
                        if (q < 3) tmem_ld32_nowait(sc + 32 * (q + 1), r[(q + 1) & 1]);
                        if (edge) {
                            const uint32_t on = seen_bits(a, i, x.n, j0 + 32 * q);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                mx4[e % 4] = fmaxf(mx4[e % 4], on >> e & 1 ? __uint_as_float(r[q & 1][e]) : -INFINITY);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e) mx4[e % 4] = fmaxf(mx4[e % 4], __uint_as_float(r[q & 1][e]));
                        }
                    }
                }
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale;
                if (W::OWN_P && !first) {
                    // P V of the block before has read the weights and written O
                    if (!(ok = warp_wait(&c.pv_done[t], (nb - 1) & 1, 111))) break;
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, mx > m + 8.f || (m == -INFINITY && mx > m))) {
                    const float n = fmaxf(m, mx), f = exp2_fast(m - (n == -INFINITY ? 0.f : n));
                    m = n;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sum[e].x *= f;
                        sum[e].y *= f;
                    }
                    if (!first) {
#pragma unroll 1
                        for (int d = 0; d < DP; d += 32) {
                            float v[32];
                            tmem_ld32(oc + d, v);
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] *= f;
                            __syncwarp();
                            tmem_st32(oc + d, v);
                        }
                    }
                }
                first = false;
                const float base = m == -INFINITY ? 0.f : m;
                {
                    uint32_t r[2][32];
                    tmem_ld32_nowait(sc, r[0]);
#pragma unroll 2
                    for (int q = 0; q < 4; ++q) {
                        tmem_wait_ld32(r[q & 1]);
                        if (q < 3) tmem_ld32_nowait(sc + 32 * (q + 1), r[(q + 1) & 1]);
                        const uint32_t on = edge ? seen_bits(a, i, x.n, j0 + 32 * q) : 0xffffffffu;
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float p0 = exp2_fast(fmaf(__uint_as_float(r[q & 1][2 * e]), a.scale, -base));
                            float p1 = exp2_fast(fmaf(__uint_as_float(r[q & 1][2 * e + 1]), a.scale, -base));
                            if (edge) {
                                p0 = on >> (2 * e) & 1 ? p0 : 0.f;
                                p1 = on >> (2 * e + 1) & 1 ? p1 : 0.f;
                            }
                            sum[e & 1] = ffma2_tc(make_float2(p0, p1), make_float2(1.f, 1.f), sum[e & 1]);
                            const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
                            pk[e] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        tmem_st16u(pc + 16 * q, pk);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&c.p_full[t]);
                ++nb;
            }
            if (!ok) break;
            if (!(ok = warp_wait(&c.pv_done[t], (nb - 1) & 1, 112))) break;
            tc_fence_after();
            const float inv = 1.f / ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
            const bool in = i < x.n;
            bool fine = true;
#pragma unroll 1
            for (int d = 0; d < DP; d += 32) {
                float v[32];
                tmem_ld32(oc + d, v);
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint4 w;
                    __nv_bfloat162* hp = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        const float y0 = in ? v[e + 2 * f] * inv : 0.f, y1 = in ? v[e + 2 * f + 1] * inv : 0.f;
                        fine = fine && isfinite(y0) && isfinite(y1);
                        hp[f] = __floats2bfloat162_rn(y0, y1);
                    }
                    if (i < a.S && d + e < a.D) *reinterpret_cast<uint4*>(o + d + e) = w;
                }
            }
            tc_fence_before();
            mbar_arrive(&c.o_empty[t]);
            for (uint32_t rows = __ballot_sync(0xffffffffu, !fine); rows; rows &= rows - 1) {
                __syncwarp();  // the row's first values are written before these
                window_row<__nv_bfloat16>(a, x.z, row0 + 32 * quad + __ffs(rows) - 1, x.h);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int DP>
int launch_window_tc(const WindowArgs& a, cudaStream_t st) {
    using W = WtShape<DP>;
    CUtensorMap tq, tk, tv;
    const uint32_t box[4] = {64, 1, 128, 1};
    auto map = [&](CUtensorMap* m, const void* p, int heads, int64_t ld) {
        const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)heads, (uint64_t)a.S, (uint64_t)a.Z};
        const uint64_t strides[3] = {(uint64_t)a.D * 2, (uint64_t)ld * 2, (uint64_t)a.S * ld * 2};
        return zg::tensor_map_bf16(m, p, 4, dims, strides, box, true);
    };
    if (!map(&tq, a.q, a.H, a.ldq) || !map(&tk, a.k, a.K, a.ldk) || !map(&tv, a.v, a.K, a.ldv))
        return zg::fail(ZG_ERR_CUDA, "zg_window_attention: tensor maps");
    if (cudaFuncSetAttribute(window_tc_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W::SMEM) !=
        cudaSuccess)
        return zg::fail(ZG_ERR_CUDA, "zg_window_attention: shared memory attribute");
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int pairs = (a.S + 255) / 256;
    const int64_t units = (int64_t)a.Z * a.H * pairs;
    zg::LaunchTimer zg_lt_("window_attention", st);
    window_tc_kernel<DP><<<(unsigned)(units < sms ? units : sms), WT_THREADS, W::SMEM, st>>>(tq, tk, tv, a, pairs, units);
    return zg::check_launch("zg_window_attention");
}

}  // namespace

namespace zg {

// Timed-out waits of the tensor-core kernel (codes 101-108, 110-112) or its
// shared memory not 1024-aligned (109); 0 = none.
int window_error_word(int clear) { return ptx_error_word(clear); }

}  // namespace zg

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
    auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if (dtype == ZG_BF16 && D <= 128 && D % 8 == 0 && ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && al(q) && al(k) &&
        al(v) && al(o) && zg::tc_available())
        return D <= 64 ? launch_window_tc<64>(a, st) : launch_window_tc<128>(a, st);
    return dtype == ZG_BF16 ? launch_window_any<__nv_bfloat16>(a, st) : launch_window_any<float>(a, st);
}
