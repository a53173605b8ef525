// zg_window.cu -- causal attention over long sequences, with a sliding window
// and a few first tokens that stay visible (sinks):
//
//   o[z, i, h] = sum_j softmax_j(q[z, i, h] . k[z, j, h / G] / sqrt(D)) v[z, j, h / G]
//   over j <= i with i - j < window or j < sinks, i, j < length[z]
//
// q, o [Z, S, H, D], k, v [Z, S, K, D], G = H / K.  Rows i >= length[z] are
// zeros.  4 D flops for each visible (i, j) and head.
#include <math.h>

#include <type_traits>

#include "zg_ptx.cuh"
#include "zg_tc.cuh"
#include "zg_warp.cuh"

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

// The larger of two values, NaN if one is.
__device__ __forceinline__ float max_nan(float x, float y) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
    return m;
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
// the tiled kernels fall back to for a row whose weights have a finite sum
// and whose outputs are not all finite.  A value of a masked place that is
// infinite or NaN has a weight of zero, and a tile's product turns 0 * inf
// into NaN; here it is not read.  (A sum that is not finite, or zero, comes
// of visible scores alone: all of the row is NaN, and stays as it is, so that
// a candidate whose activations are all NaN costs nothing here.)
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
    // four positions at a time, their reads in flight together
    for (int j0 = 0; j0 <= i; j0 += 4) {
        if (!sees(a, i, j0) && !sees(a, i, j0 + 3 < i ? j0 + 3 : i)) {
            j0 = i - a.window - 3;  // the window's first position is next
            continue;
        }
        float s[4], n = m;
        bool on[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            on[g] = j0 + g <= i && sees(a, i, j0 + g);
            s[g] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = lane + 32 * e;
                if (on[g] && d < a.D) s[g] = fmaf(qv[e], zg_to_float(k[(j0 + g) * a.ldk + d]), s[g]);
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
            for (int f = 16; f > 0; f >>= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], f);
            s[g] = on[g] ? s[g] : -INFINITY;
            n = fmaxf(n, s[g]);
        }
        const float base = n == -INFINITY ? 0.f : n, c = exp2f(m - base);
        l *= c;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= c;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float p = exp2f(s[g] - base);
            l += p;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = lane + 32 * e;
                if (on[g] && d < a.D) x[e] = fmaf(p, zg_to_float(v[(j0 + g) * a.ldv + d]), x[e]);
            }
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
// A block has 32 query rows of one head and walks over the tiles of 64 keys
// that any of them sees, q, k, v and the weights in shared memory as float32.
// 128 threads as 8 x 16: thread (ty, tx) has the scores of rows ty + 8 i
// and keys tx + 16 j, and the outputs of the same rows in column pairs
// 2 tx + 32 c.  Both products are in packed pairs (two FMAs an instruction):
// of the scores the even and the odd columns' sums apart, of the outputs two
// columns.  Rows are DP + 4 floats apart, so that the 16-byte reads of
// neighbouring rows fall into different banks.  Float32 rows come by cp.async,
// the next tile's keys under this one's second product and its values under
// the next first one; others are converted on the way, a tile's words in
// flight together.  Of a tile at the edge of the mask only those sixteens of
// keys are multiplied that any row sees: 3 x 777 tokens of 8 heads of 80 under
// a window of 200, 65 -> 52 us.  What bounds it is the FMA pipe and the shared
// memory reads that feed it, both over half busy: causal, 2048 tokens of 8
// heads of 128, 269 us, 32 TFLOP/s of the visible pairs.
// ---------------------------------------------------------------------------
constexpr int WF_M = 32, WF_N = 64, WF_THREADS = 128, WF_PP = WF_N + 4;

template <int DP>
constexpr size_t wf_smem() {
    return (size_t)((WF_M + 2 * WF_N) * (DP + 4) + WF_M * WF_PP) * sizeof(float);
}

template <typename T, int DP>
__global__ void __launch_bounds__(WF_THREADS, DP <= 96 ? 3 : DP <= 128 ? 2 : 1) window_fma_kernel(const WindowArgs a, int q_tiles, int vec) {
    constexpr int PITCH = DP + 4, NC = DP / 32;
    extern __shared__ __align__(16) float sm[];
    float *qs = sm, *ks = qs + WF_M * PITCH, *vs = ks + WF_N * PITCH, *ps = vs + WF_N * PITCH;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    // the tiles that see the most keys first, of all heads: 2048 tokens of 8
    // heads of 128 are 256 blocks of 1 to 32 tiles (head by head the SMs
    // were busy for 61% of the time)
    const int heads = a.Z * a.H;
    const int qt = q_tiles - 1 - (int)(blockIdx.x / heads), zh = (int)(blockIdx.x % heads);
    const int z = zh / a.H, h = zh % a.H, kh = h / a.G;
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

    // ROWS rows from r0, zeros past n and D
    auto load = [&](auto rows, float* dst, const T* src, int64_t ld, int r0) {
        constexpr int ROWS = decltype(rows)::value;
        constexpr int WORDS = DP / 4, EACH = ROWS * WORDS / WF_THREADS;  // 16-byte words of a row, words of a thread
        if (sizeof(T) == 4 && vec) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int x = threadIdx.x + e * WF_THREADS, r = x / WORDS, d = x % WORDS * 4;
                const bool on = r0 + r < n && d < a.D;
                copy16(smem_u32(dst + r * PITCH + d), on ? src + (r0 + r) * ld + d : src, on ? 16 : 0);
            }
        } else if (vec) {
            uint2 u[EACH];
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int x = threadIdx.x + e * WF_THREADS, r = x / WORDS, d = x % WORDS * 4;
                u[e] = r0 + r < n && d < a.D ? *reinterpret_cast<const uint2*>(src + (r0 + r) * ld + d) : make_uint2(0, 0);
            }
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int x = threadIdx.x + e * WF_THREADS, r = x / WORDS, d = x % WORDS * 4;
                *reinterpret_cast<float4*>(dst + r * PITCH + d) =
                    make_float4(__uint_as_float(u[e].x << 16), __uint_as_float(u[e].x & 0xffff0000u),
                                __uint_as_float(u[e].y << 16), __uint_as_float(u[e].y & 0xffff0000u));
            }
        } else {
#pragma unroll 8
            for (int x = threadIdx.x; x < ROWS * DP; x += WF_THREADS) {
                const int r = x / DP, d = x % DP;
                dst[r * PITCH + d] = r0 + r < n && d < a.D ? zg_to_float(src[(r0 + r) * ld + d]) : 0.f;
            }
        }
        copy_commit();
    };
    const std::integral_constant<int, WF_M> q_rows{};
    const std::integral_constant<int, WF_N> k_rows{};
    load(q_rows, qs, q, a.ldq, i0);

    const float2 zero2 = make_float2(0.f, 0.f);
    float2 x[4][NC];
    float m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) x[i][c] = zero2;
    }
    const int last = i0 + WF_M < n ? i0 + WF_M : n;  // rows [i0, last)
    const int kt_end = (last + WF_N - 1) / WF_N;
    const int w0 = i0 - a.window + 1 > 0 ? (i0 - a.window + 1) / WF_N : 0;  // the window's first tile
    int sink_end = (a.sinks + WF_N - 1) / WF_N;                              // tiles that hold sinks
    if (sink_end > w0) sink_end = w0;
    auto next = [&](int kt) { return kt + 1 < sink_end || kt >= w0 ? kt + 1 : w0; };
    int kt = sink_end > 0 ? 0 : w0;
    load(k_rows, ks, k, a.ldk, kt * WF_N);
    for (; kt < kt_end; kt = next(kt)) {
        const int j0 = kt * WF_N;
        load(k_rows, vs, v, a.ldv, j0);
        copy_wait<1>();  // the keys
        __syncthreads();
        // the sixteens of this tile's keys that any row sees: [g0, g1)
        int lo = i0 - a.window + 1 - j0, hi = last - j0;
        if (lo <= 0 || j0 < a.sinks) lo = 0;
        if (i0 - a.window + 1 - j0 >= WF_N) hi = a.sinks - j0;  // sinks alone
        const int g0 = lo / 16, g1 = hi >= WF_N ? 4 : (hi + 15) / 16;
        // the scores of NG sixteens, and their softmax into ps
        auto scores = [&](auto groups) {
            constexpr int NG = decltype(groups)::value;
            const float* kr = ks + (16 * g0 + tx) * PITCH;
            float2 s2[4][NG];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NG; ++j) s2[i][j] = zero2;
#pragma unroll 2
            for (int d = 0; d < DP; d += 4) {
                float4 qv[4], kv[NG];
#pragma unroll
                for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(qs + (ty + 8 * i) * PITCH + d);
#pragma unroll
                for (int j = 0; j < NG; ++j) kv[j] = *reinterpret_cast<const float4*>(kr + 16 * j * PITCH + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        s2[i][j] = ffma2_tc(make_float2(qv[i].x, qv[i].y), make_float2(kv[j].x, kv[j].y), s2[i][j]);
                        s2[i][j] = ffma2_tc(make_float2(qv[i].z, qv[i].w), make_float2(kv[j].z, kv[j].w), s2[i][j]);
                    }
            }
            copy_wait<0>();  // the values
            __syncthreads();
            if (next(kt) < kt_end)
                load(k_rows, ks, k, a.ldk, next(kt) * WF_N);
            else
                copy_commit();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int qi = i0 + ty + 8 * i;
                float s[NG], t = m[i];
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const int kj = j0 + 16 * (g0 + j) + tx;
                    s[j] = kj <= qi && kj < n && sees(a, qi, kj) ? (s2[i][j].x + s2[i][j].y) * a.scale : -INFINITY;
                    t = fmaxf(t, s[j]);
                }
#pragma unroll
                for (int f = 8; f > 0; f >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, f));
                const float base = t == -INFINITY ? 0.f : t;
                const float c = exp2f(m[i] - base);
                m[i] = t;
                l[i] *= c;
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const float p = exp2f(s[j] - base);
                    l[i] += p;
                    ps[(ty + 8 * i) * WF_PP + 16 * (g0 + j) + tx] = p;
                }
#pragma unroll
                for (int e = 0; e < NC; ++e) x[i][e] = ffma2_tc(x[i][e], make_float2(c, c), zero2);
            }
        };
        switch (g1 - g0) {
            case 4: scores(std::integral_constant<int, 4>{}); break;
            case 3: scores(std::integral_constant<int, 3>{}); break;
            case 2: scores(std::integral_constant<int, 2>{}); break;
            default: scores(std::integral_constant<int, 1>{});
        }
        __syncwarp();  // a row's weights are written and read by the same half warp
#pragma unroll 4
        for (int j = 16 * g0; j < 16 * g1; j += 4) {
            float4 pv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = *reinterpret_cast<const float4*>(ps + (ty + 8 * i) * WF_PP + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float2 vv = *reinterpret_cast<const float2*>(vs + (j + e) * PITCH + 32 * c + 2 * tx);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = e == 0 ? pv[i].x : e == 1 ? pv[i].y : e == 2 ? pv[i].z : pv[i].w;
                        x[i][c] = ffma2_tc(make_float2(p, p), vv, x[i][c]);
                    }
                }
            }
        }
        __syncthreads();  // the values have been read
    }
    unsigned redo = 0;  // bit i: row i of this half warp is formed again
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int f = 8; f > 0; f >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], f);
        const int qi = i0 + ty + 8 * i;
        bool fine = true;
        const bool known = l[i] > 0.f && l[i] < INFINITY;  // else all NaN, by its visible scores
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = 32 * c + 2 * tx + e;
                const float y = qi < n ? (e ? x[i][c].y : x[i][c].x) / l[i] : 0.f;
                if (d < a.D) {
                    fine = fine && isfinite(y);
                    if (qi < a.S) o[qi * ldo + d] = zg_from_float<T>(y);
                }
            }
        const unsigned half = 0xffffu << (threadIdx.x % 32 / 16 * 16);
        if (__ballot_sync(0xffffffffu, known && !fine) & half) redo |= 1u << i;
    }
    // the rows of this warp's two halves, one at a time by the whole warp
    for (int t = 0; t < 2; ++t) {
        const unsigned rows = __shfl_sync(0xffffffffu, redo, 16 * t);
        for (int i = 0; i < 4; ++i)
            if (rows >> i & 1) {
                __syncwarp();  // the row's first values are written before these
                window_row<T>(a, z, i0 + (int)(threadIdx.x / 32) * 2 + t + 8 * i, h);
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
    return a.D <= 32    ? launch_window_fma<T, 32>(a, vec, st)
           : a.D <= 64  ? launch_window_fma<T, 64>(a, vec, st)
           : a.D <= 96  ? launch_window_fma<T, 96>(a, vec, st)
           : a.D <= 128 ? launch_window_fma<T, 128>(a, vec, st)
           : a.D <= 192 ? launch_window_fma<T, 192>(a, vec, st) : launch_window_fma<T, 256>(a, vec, st);
}

// ---------------------------------------------------------------------------
// Tensor-core path: bf16, D <= DP (64 or 128, zeros behind D).
//
// A CTA per SM, which takes unit after unit, 384 threads: warp 0 issues the TMA loads, warps
// 1 and 2 the MMAs of a tile each, warps 4-7 and 8-11 are the softmax groups
// of two tiles of 128 query rows (one thread a row); warp 3 fills the group of
// four that setmaxnreg speaks to.  A work unit is a pair of neighbouring tiles
// of one (z, head), so that each block of keys and values is fetched once for
// both; the units with the most visible keys come first.  Per block and tile:
// S = Q K^T into TMEM (M = 128, N = KEYS), a row's maximum, the weights
// p = 2^(s - m) as bf16 back into TMEM, O += P V with P read from TMEM.  Only
// blocks that a tile sees any key of are visited, and only those at the edge
// of a warp's mask test each key.
//
// TMEM (512 columns): O of the two tiles, and of each tile one buffer of
// scores and weights of their own columns: with DP = 64 blocks of 128 keys
// (128 + 64 columns), with DP = 128, where O takes twice as much, blocks of 64
// keys and two buffers of weights (64 + 2 * 32).  A group reads a block's
// scores into registers and says so, and the next block's Q K^T runs under its
// softmax; the weights do not hold it up.  (Weights over the scores they came
// from, the next Q K^T behind P V: 2100 clocks a block of 64 at D = 128, 600 of
// them waiting for scores.  Blocks of 64 keys at D = 64: each block's signals
// between the roles cost what its exponentials do.)
//
// What bounds it is a group's exponentials, 16 a clock and SM, and the waits
// around them; the MMAs take about half as long.  2 x 4096 tokens of 12 heads
// (4 key heads) of 64, causal: 82 us, 0.62 PFLOP/s of the visible pairs; 8192
// tokens of 16 heads (4) of 128 under a window of 1024: 87 us, 0.74 PFLOP/s.
//
// The maximum m that weights are taken against is moved, and O rescaled by
// its group, only when a row's true maximum is more than 2^8 above it: the
// quotient O / l is the same, weights stay below 2^8 (and their relative
// rounding in bf16 is what it was), and after the first blocks O is hardly
// ever touched.
// ---------------------------------------------------------------------------
constexpr int WT_THREADS = 384;

template <int DP>
struct WtShape {
    static constexpr int KEYS = DP == 64 ? 128 : 64;         // keys of a block
    static constexpr uint32_t QTILE = 128 * DP * 2;          // a query tile: DP / 64 boxes of 128 rows x 64 columns
    static constexpr uint32_t BOX = KEYS * 128;              // KEYS rows x 64 columns
    static constexpr uint32_t BLOCK = KEYS * DP * 2;         // a key or value block: DP / 64 boxes
    static constexpr int STAGES = 5;                         // ring of blocks, the keys and behind them the values
    static constexpr uint32_t RING = 2 * QTILE;
    static constexpr uint32_t CTRL = RING + STAGES * 2 * BLOCK;
    static constexpr uint32_t SMEM = CTRL + 512;
    static constexpr uint32_t PB = DP == 64 ? 1 : 2;         // buffers of weights of a tile
    static constexpr uint32_t TILE_COLS = KEYS + PB * (KEYS / 2);
    // TMEM columns of tile t's scores, of its weights of block n, and of its outputs
    static __device__ __forceinline__ uint32_t s_col(int t) { return t * TILE_COLS; }
    static __device__ __forceinline__ uint32_t p_col(int t, uint32_t n) { return t * TILE_COLS + KEYS + n % PB * (KEYS / 2); }
    static __device__ __forceinline__ uint32_t o_col(int t) { return 2 * TILE_COLS + t * DP; }
    static_assert(2 * TILE_COLS + 2 * DP == 512, "all of TMEM");
};

// With two buffers of weights a warp of a group may be a block ahead of the
// others (never two: the scores after next wait until all have read the next
// ones), so each has a barrier; and that a block's scores are there says, by
// the order of the issuer's commits, that P V of two blocks before is done.
// With one buffer a group waits for P V of the block before.
struct alignas(16) WtCtrl {
    uint4 unit[4];  // answers to the requests for the next unit
    uint64_t unit_full[4], unit_empty[4];
    uint64_t q_full[2], q_empty[2], kv_full[5], kv_empty[5], s_full[2], s_read[2], p_full[2][2], pv_done[2], o_full[2], o_empty[2], done;
    uint32_t tmem_base;
    int redo[8];  // of each softmax warp: the last unit with rows to be formed again
};
static_assert(sizeof(WtCtrl) <= 512, "control block");

// What stands in column 0 of a row that is to be formed again: a NaN that no
// rounding gives.  Columns 2 and 3 hold the warp's unit before with such rows.
constexpr uint16_t WT_REDO = 0x7fa5;

// A unit as the role of tile t sees it: two tiles of 128 rows from i0, the
// blocks of keys that either sees (first .. hi, next() from one to the next)
// and those that this tile does.
struct WtUnit {
    int z, h, n, i0, sink_blocks, lo0, hi;
    int lo, last;  // the first block of this tile's window, and its last (-1: a tile behind the sequence)
    bool any, both;  // whether the sequence reaches the first tile, and the second
    __device__ __forceinline__ bool takes(int b) const { return b <= last && (b >= lo || b < sink_blocks); }
    __device__ __forceinline__ int first() const { return sink_blocks > 0 ? 0 : lo0; }
    __device__ __forceinline__ int next(int b) const { return b + 1 < sink_blocks || b + 1 >= lo0 ? b + 1 : lo0; }
};

template <int KEYS>
__device__ __forceinline__ WtUnit wt_unit(const WindowArgs& a, int u, int pairs, int t) {
    WtUnit x;
    const int heads = a.Z * a.H, pair = pairs - 1 - u / heads, zh = u % heads;
    x.z = zh / a.H;
    x.h = zh % a.H;
    x.n = length_of(a, x.z);
    x.i0 = pair * 256;
    x.any = x.i0 < x.n;
    x.both = x.i0 + 128 < x.n;
    x.sink_blocks = (a.sinks + KEYS - 1) / KEYS;
    const int w0 = x.i0 - a.window + 1, w = w0 + 128 * t;
    x.lo0 = w0 > 0 ? w0 / KEYS : 0;
    x.lo = w > 0 ? w / KEYS : 0;
    const int end = x.i0 + 256 < x.n ? x.i0 + 256 : x.n, mine = x.i0 + 128 * (t + 1);
    x.hi = (end - 1) / KEYS;
    x.last = (t ? x.both : x.any) ? ((mine < x.n ? mine : x.n) - 1) / KEYS : -1;
    return x;
}

// Units are the blocks of the grid, and a CTA that has taken one asks for the
// next that no CTA has started, so that the CTAs end together whatever the
// sequences' lengths are.  (Units dealt out beforehand, in rows there and back,
// against this: 2 x 4096 causal 95 -> 83 us; 8192 under a window of 1024 102 ->
// 87 us; 16 padded sequences of up to 1000 under a window of 100 52 -> 42 us.)
// The loader asks, and every role reads the answer.
__device__ __forceinline__ void unit_request(uint4* to, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(to)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// The unit of an answer, -1 when there is none left.
__device__ __forceinline__ int unit_answer(const uint4* from) {
    int u;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
        "ld.shared.b128 h, [%1];\n\t"
        "mov.b32 %0, -1;\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}"
        : "=r"(u)
        : "r"(smem_u32(from))
        : "memory");
    return u;
}

// Bits 0 .. x of a word.
__device__ __forceinline__ uint32_t bits_upto(int x) { return x < 0 ? 0u : x >= 31 ? 0xffffffffu : (2u << x) - 1u; }

// The keys jc .. jc + 31 that row i of a sequence of n sees, as bits.
__device__ __forceinline__ uint32_t seen_bits(const WindowArgs& a, int i, int n, int jc) {
    const int last = i < n - 1 ? i : n - 1;
    return bits_upto(last - jc) & (~bits_upto(i - a.window - jc) | bits_upto(a.sinks - 1 - jc));
}

// Whether a phase has completed, without waiting for it.
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}

// The unit that follows a role's k-th: -1 for none, or when the wait ran out.
__device__ __forceinline__ int unit_after(WtCtrl& c, uint32_t k, bool& ok) {
    if (!ok || !(ok = warp_wait(&c.unit_full[k % 4], (k / 4) & 1, 109))) return -1;
    const int u = unit_answer(&c.unit[k % 4]);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (threadIdx.x % 32 == 0) mbar_arrive(&c.unit_empty[k % 4]);
    return __shfl_sync(0xffffffffu, u, 0);
}

// MMAs and commits issued by one elected lane of a converged warp, always the
// same one.  The warp walks its blocks together, so that addresses and
// descriptors are uniform values: a role entered by lane 0 alone had each
// operand moved over for each instruction, 70 clocks an MMA.
__device__ __forceinline__ void umma_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_ts_elect(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_commit_elect(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}

template <int DP>
__global__ void __launch_bounds__(WT_THREADS, 1)
window_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const WindowArgs a, int pairs) {
    using W = WtShape<DP>;
    // No static shared memory, so the dynamic block starts at the CTA's first
    // shared byte; the swizzled tiles need it 1024-aligned, which is checked.
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicCAS(&g_zg_tc_error, 0u, 110u);
        return;
    }
    WtCtrl& c = *reinterpret_cast<WtCtrl*>(smem + W::CTRL);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    if (threadIdx.x < 8) c.redo[threadIdx.x] = -1;
    if (threadIdx.x == 0) {
        mbar_init(&c.done, 2);  // both issuers
        for (int i = 0; i < 4; ++i) {
            mbar_init(&c.unit_full[i], 1);
            mbar_init(&c.unit_empty[i], 10);  // the issuers and the softmax warps
        }
        for (int i = 0; i < W::STAGES; ++i) {
            mbar_init(&c.kv_full[i], 1);
            mbar_init(&c.kv_empty[i], 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&c.q_full[t], 1);
            mbar_init(&c.q_empty[t], 1);
            mbar_init(&c.s_full[t], 1);
            for (int i = 0; i < 2; ++i) mbar_init(&c.p_full[t][i], 128);
            mbar_init(&c.s_read[t], 128);
            mbar_init(&c.pv_done[t], 1);
            mbar_init(&c.o_full[t], 1);
            mbar_init(&c.o_empty[t], 128);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(&c.tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = c.tmem_base;

    // A softmax thread holds a block's scores: the launch's 384 x 168
    // registers are shared out as 128 x 72 and 256 x 216.
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
        if (lane == 0) {
            // blocks and query tiles loaded; a stage's parity follows from the count
            uint32_t nk = 0, nq[2] = {0, 0}, nr = 0;
            bool ok = true;
            // the next unit, asked for when this one's blocks are on their way
            auto request = [&]() {
                uint64_t* full = &c.unit_full[nr % 4];
                if (!ok || !(ok = mbar_wait(&c.unit_empty[nr % 4], ((nr / 4) & 1) ^ 1, 114))) return -1;
                mbar_expect_tx(full, 16);
                unit_request(&c.unit[nr % 4], full);
                if (!(ok = mbar_wait(full, (nr / 4) & 1, 115))) return -1;
                return unit_answer(&c.unit[nr++ % 4]);
            };
            for (int u = blockIdx.x; u >= 0; u = request()) {
                const WtUnit x = wt_unit<W::KEYS>(a, u, pairs, 0);
                if (!x.any) continue;
                const int kh = x.h / a.G;
                auto queries = [&](int t) {
                    if (!mbar_wait(&c.q_empty[t], (nq[t] & 1) ^ 1, 101)) return false;
                    mbar_expect_tx(&c.q_full[t], W::QTILE);
                    for (int d = 0; d < DP / 64; ++d)
                        tma_load_4d(smem + t * W::QTILE + d * 16384, &tmQ, &c.q_full[t], 64 * d, x.h, x.i0 + 128 * t, x.z);
                    ++nq[t];
                    return true;
                };
                if (!(ok = queries(0))) break;
                // The second tile's queries come two blocks later: the first tile
                // may be that far into its unit while the second ends its last.
                int ahead = x.both ? 2 : -1;
                for (int b = x.first(); b <= x.hi; b = x.next(b), ++nk) {
                    if (ahead >= 0 && ahead-- == 0 && !(ok = queries(1))) break;
                    const uint32_t st = nk % W::STAGES;
                    if (!(ok = mbar_wait(&c.kv_empty[st], ((nk / W::STAGES) & 1) ^ 1, 102))) break;
                    mbar_expect_tx(&c.kv_full[st], 2 * W::BLOCK);
                    for (int d = 0; d < DP / 64; ++d) {
                        uint8_t* to = smem + W::RING + st * 2 * W::BLOCK + d * W::BOX;
                        tma_load_4d(to, &tmK, &c.kv_full[st], 64 * d, kh, b * W::KEYS, x.z);
                        tma_load_4d(to + W::BLOCK, &tmV, &c.kv_full[st], 64 * d, kh, b * W::KEYS, x.z);
                    }
                }
                if (ok && ahead >= 0) ok = queries(1);  // a unit of two blocks or fewer
            }
            // loads still in flight (only after an abort) land before the CTA exits
            for (uint32_t s = nk > W::STAGES ? nk - W::STAGES : 0; s < nk; ++s)
                for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&c.kv_full[s % W::STAGES], (s / W::STAGES) & 1); ++i) {
                }
            for (int t = 0; t < 2; ++t)
                if (nq[t])
                    for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&c.q_full[t], (nq[t] - 1) & 1); ++i) {
                    }
        }
    } else if (warp <= 2) {
        // one MMA issuer per tile; both give every block back to the loader
        const int t = warp - 1;
        const uint32_t idesc_s = idesc_bf16(128, W::KEYS, 0), idesc_o = idesc_bf16(128, DP, 1);
        const uint32_t qa = smem_u32(smem + t * W::QTILE), ring = smem_u32(smem + W::RING);
        uint32_t nk = 0, ns = 0, npv = 0, nu = 0, taken = 0;  // blocks, and of this tile scores, outputs, units
        bool ok = true;
        for (int u = blockIdx.x; u >= 0; u = unit_after(c, taken++, ok)) {
            const WtUnit x = wt_unit<W::KEYS>(a, u, pairs, t);
            if (!x.any) continue;
            if (x.last >= 0 && !(ok = warp_wait(&c.q_full[t], nu & 1, 103))) break;
            bool started = false;
            bool pending = false;  // P V of the last scores is to come
            uint32_t vstage = 0;   // with the values of this stage
            int vblock = -1;       // and the number of their block
            auto outputs = [&]() {
                const uint32_t st = vstage;
                const uint32_t va = ring + st * 2 * W::BLOCK + W::BLOCK;
                if (x.n < a.S && (vblock + 1) * W::KEYS > x.n) {
                    // rows of a padded batch behind this sequence: their weights are
                    // zeros, and so are their values then, whatever they hold
                    const uint32_t r0 = (uint32_t)(x.n - vblock * W::KEYS) * 128u;
                    for (int d = 0; d < DP / 64; ++d)
                        for (uint32_t at = r0 + lane * 16; at < W::BOX; at += 512)
                            *reinterpret_cast<uint4*>(smem + (va - smem_u32(smem)) + d * W::BOX + at) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (!warp_wait(&c.p_full[t][npv & 1], (npv >> 1) & 1, 104)) return false;
                // the last unit's outputs have been read
                if (!started && !warp_wait(&c.o_empty[t], (nu & 1) ^ 1, 105)) return false;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < W::KEYS / 16; ++k)
                    umma_ts_elect(tmem + W::o_col(t), tmem + W::p_col(t, npv) + k * 8, smem_desc(va + k * 2048, W::BOX, 1024),
                                  idesc_o, started || k > 0 ? 1u : 0u);
                umma_commit_elect(&c.pv_done[t]);
                if (vblock == x.last) umma_commit_elect(&c.o_full[t]);
                umma_commit_elect(&c.kv_empty[st]);
                ++npv;
                started = true;
                pending = false;
                return true;
            };
            for (int b = x.first(); b <= x.hi; b = x.next(b), ++nk) {
                const uint32_t st = nk % W::STAGES, parity = (nk / W::STAGES) & 1;
                if (!x.takes(b)) {
                    if (pending) ok = outputs();
                    // a block that is the other tile's alone is given back once it is here
                    if (!ok || !(ok = warp_wait(&c.kv_full[st], parity, 106))) break;
                    if (lane == 0) mbar_arrive(&c.kv_empty[st]);
                    __syncwarp();
                    continue;
                }
                if (!(ok = warp_wait(&c.kv_full[st], parity, 107))) break;
                // the last scores are in their rows' registers
                if (ns > 0 && !(ok = warp_wait(&c.s_read[t], (ns - 1) & 1, 108))) break;
                tc_fence_after();
                const uint32_t ka = ring + st * 2 * W::BLOCK;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
                    umma_elect(tmem + W::s_col(t), smem_desc(qa + (k / 4) * 16384 + (k % 4) * 32, 16, 1024),
                               smem_desc(ka + (k / 4) * W::BOX + (k % 4) * 32, 16, 1024), idesc_s, k > 0 ? 1u : 0u);
                umma_commit_elect(&c.s_full[t]);
                if (b == x.last) umma_commit_elect(&c.q_empty[t]);
                ++ns;
                if (pending && !(ok = outputs())) break;
                pending = true;
                vstage = st;
                vblock = b;
            }
            if (!ok || (pending && !(ok = outputs()))) break;
            if (started) ++nu;
        }
        // every MMA this thread issued has completed before TMEM is freed
        umma_commit_elect(&c.done);
        for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&c.done, 0); ++i) {
        }
    } else if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int t = (warp - 4) / 4, quad = warp % 4;
        const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t oc = trow + W::o_col(t);
        const int64_t ldo = (int64_t)a.H * a.D;
        const float2 one2 = make_float2(1.f, 1.f), scale2 = make_float2(a.scale, a.scale);
        uint32_t nb = 0, nu = 0, taken = 0;  // blocks and units of this tile so far, units of both
        bool s_ready = false;                // the next scores have been seen to be there
        bool ok = true;
        for (int u = blockIdx.x; u >= 0; u = unit_after(c, taken++, ok)) {
            const WtUnit x = wt_unit<W::KEYS>(a, u, pairs, t);
            const int row0 = x.i0 + 128 * t + 32 * quad, i = row0 + lane;  // the warp's first row, this thread's
            __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.o) + ((int64_t)x.z * a.S + i) * ldo + (int64_t)x.h * a.D;
            if (x.last < 0) {
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
                if (!x.takes(b)) continue;
                const uint32_t sc = trow + W::s_col(t), pc = trow + W::p_col(t, nb);
                if (!s_ready && !(ok = warp_wait(&c.s_full[t], nb & 1, 111))) break;
                tc_fence_after();
                const int j0 = b * W::KEYS;
                // The maximum m is moved to the row's (mx, scaled) where that is more
                // than 2^8 above; false when a wait ran out.
                auto settle = [&](float mx, bool pv_seen) {
                    // P V of the block before has read the weights' buffer and added to O
                    const bool all_seen = __all_sync(0xffffffffu, pv_seen);
                    if (W::PB == 1 && !first) {
                        if (!all_seen && !warp_wait(&c.pv_done[t], (nb - 1) & 1, 112)) return false;
                        tc_fence_after();
                    }
                    if (!__any_sync(0xffffffffu, i < x.n && !(mx <= m + 8.f))) return true;  // rows behind the sequence do not count
                    const float n = fmaxf(m, mx);
                    float f = exp2_fast(m - (n == -INFINITY ? 0.f : n));
                    // a score that is NaN or infinite: the row is formed again at the end
                    if (!(mx < INFINITY)) f = __int_as_float(0x7fffffff);
                    m = n;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sum[e].x *= f;
                        sum[e].y *= f;
                    }
                    if (first) return true;
                    if (W::PB == 2) {
                        if (!all_seen && !warp_wait(&c.pv_done[t], (nb - 1) & 1, 112)) return false;
                        tc_fence_after();
                    }
#pragma unroll 1
                    for (int d = 0; d < DP; d += 32) {
                        float v[32];
                        tmem_ld32(oc + d, v);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] *= f;
                        __syncwarp();
                        tmem_st32(oc + d, v);
                    }
                    return true;
                };
                // whether every row of this warp sees all of the block, or any row any of keys jc ..
                const bool full = j0 + W::KEYS - 1 <= row0 && (j0 > row0 + 31 - a.window || j0 + W::KEYS <= a.sinks);
                auto seen = [&](int jc, int keys) {
                    return jc <= row0 + 31 && (jc + keys - 1 > row0 - a.window || jc < a.sinks);
                };
                if (W::KEYS == 64 && !seen(j0, 64)) {
                    mbar_arrive(&c.s_read[t]);
                    uint32_t zero[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) zero[e] = 0u;
                    tmem_st16u(pc, zero);
                    tmem_st16u(pc + 16, zero);
                } else if (full || W::KEYS == 64) {
                    // a row's scores stay in its thread's registers
                    uint32_t r[W::KEYS / 32][32];
#pragma unroll
                    for (int q = 0; q < W::KEYS / 32; ++q) tmem_ld32_nowait(sc + 32 * q, r[q]);
#pragma unroll
                    for (int q = 0; q < W::KEYS / 32; ++q) tmem_wait_ld32(r[q]);
                    tc_fence_before();
                    mbar_arrive(&c.s_read[t]);
                    // asked now, used behind the maximum: an answer takes some 250 clocks
                    // behind the exponentials in the same queue
                    const bool pv_seen = !first && mbar_test_wait(&c.pv_done[t], (nb - 1) & 1);
                    if (W::KEYS == 64 && !full) {
                        // keys that the row does not see score -inf
#pragma unroll
                        for (int q = 0; q < W::KEYS / 32; ++q) {
                            const uint32_t on = seen_bits(a, i, x.n, j0 + 32 * q);
#pragma unroll
                            for (int e = 0; e < 32; ++e) r[q][e] = on >> e & 1 ? r[q][e] : 0xff800000u;
                        }
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int q = 0; q < W::KEYS / 32; q += 2)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            mx4[e % 4] = max_nan(mx4[e % 4], max_nan(__uint_as_float(r[q][e]), __uint_as_float(r[q + 1][e])));
                    const float mx = max_nan(max_nan(mx4[0], mx4[1]), max_nan(mx4[2], mx4[3])) * a.scale;
                    if (!(ok = settle(mx, pv_seen))) break;
                    const float base = m == -INFINITY ? 0.f : m;
                    const float2 base2 = make_float2(-base, -base);
#pragma unroll
                    for (int q = 0; q < W::KEYS / 32; ++q) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float2 y = ffma2_tc(
                                make_float2(__uint_as_float(r[q][2 * e]), __uint_as_float(r[q][2 * e + 1])), scale2, base2);
                            const float2 w = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                            sum[e & 1] = ffma2_tc(w, one2, sum[e & 1]);
                            const __nv_bfloat162 v = __floats2bfloat162_rn(w.x, w.y);
                            pk[e] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        tmem_st16u(pc + 16 * q, pk);
                    }
                } else {
                    // The mask cuts a block of 128: 32 keys at a time, read twice, those that no
                    // row of the warp sees passed over, and those that all rows see not masked
                    // (16 x 256 under a window of 64: 16.3 -> 15.5 us).  With the mask in the
                    // path above D = 64 was 10% slower; two paths of 128 registers each spill.
                    // At D = 128, with 64, one path with the mask in it is 7% faster under a
                    // window of 1024, and leaving out the 32 keys that no row sees 3% slower.
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int q = 0; q < W::KEYS / 32; ++q) {
                        const int jc = j0 + 32 * q;
                        if (!seen(jc, 32)) continue;
                        float v[32];
                        tmem_ld32(sc + 32 * q, v);
                        const uint32_t on = seen_bits(a, i, x.n, jc);
                        if (!__all_sync(0xffffffffu, on == ~0u)) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = on >> e & 1 ? v[e] : -INFINITY;
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) mx4[e % 4] = max_nan(mx4[e % 4], v[e]);
                    }
                    const float mx = max_nan(max_nan(mx4[0], mx4[1]), max_nan(mx4[2], mx4[3]));
                    const bool pv_seen = !first && mbar_test_wait(&c.pv_done[t], (nb - 1) & 1);
                    if (!(ok = settle(mx * a.scale, pv_seen))) break;
                    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 1
                    for (int q = 0; q < W::KEYS / 32; ++q) {
                        const int jc = j0 + 32 * q;
                        uint32_t pk[16];
                        if (seen(jc, 32)) {
                            float v[32];
                            tmem_ld32(sc + 32 * q, v);
                            const uint32_t on = seen_bits(a, i, x.n, jc);
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = exp2_fast(fmaf(v[e], a.scale, -base));
                            if (!__all_sync(0xffffffffu, on == ~0u)) {
#pragma unroll
                                for (int e = 0; e < 32; ++e) v[e] = on >> e & 1 ? v[e] : 0.f;
                            }
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                sum[e & 1] = ffma2_tc(make_float2(v[2 * e], v[2 * e + 1]), one2, sum[e & 1]);
                                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                                pk[e] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) pk[e] = 0u;
                        }
                        tmem_st16u(pc + 16 * q, pk);
                    }
                    tc_fence_before();
                    mbar_arrive(&c.s_read[t]);
                }
                // whether the next scores are there, asked while the stores go
                const bool next_ready = mbar_test_wait(&c.s_full[t], (nb + 1) & 1);
                first = false;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&c.p_full[t][nb & 1]);
                ++nb;
                s_ready = __all_sync(0xffffffffu, next_ready);
            }
            if (!ok) break;
            if (!(ok = warp_wait(&c.o_full[t], nu & 1, 113))) break;
            ++nu;
            tc_fence_after();
            const float l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), inv = 1.f / l;
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
            const bool again = !fine && l > 0.f && l < INFINITY;
            if (__any_sync(0xffffffffu, again)) {
                int* before = &c.redo[warp - 4];
                if (again) {
                    *reinterpret_cast<uint16_t*>(o) = WT_REDO;
                    *reinterpret_cast<int*>(o + 2) = *before;
                }
                __syncwarp();
                if (lane == 0) *before = u;
                __syncwarp();
            }
        }
        // The marked rows, the last unit's first, when no role waits for this one
        // any more: a row of 10^5 keys takes longer than the waits' limit.
        for (int u = ok ? c.redo[warp - 4] : -1; u >= 0;) {
            const WtUnit x = wt_unit<W::KEYS>(a, u, pairs, t);
            const int row0 = x.i0 + 128 * t + 32 * quad, i = row0 + lane;
            const __nv_bfloat16* o = static_cast<const __nv_bfloat16*>(a.o) + ((int64_t)x.z * a.S + i) * ldo + (int64_t)x.h * a.D;
            const bool again = i < x.n && *reinterpret_cast<const uint16_t*>(o) == WT_REDO;
            const int before = again ? *reinterpret_cast<const int*>(o + 2) : -1;
            uint32_t rows = __ballot_sync(0xffffffffu, again);
            u = __shfl_sync(0xffffffffu, before, __ffs(rows) - 1);
            for (; rows; rows &= rows - 1) window_row<__nv_bfloat16>(a, x.z, row0 + __ffs(rows) - 1, x.h);
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
    auto map = [&](CUtensorMap* m, const void* p, int heads, int64_t ld, uint32_t rows) {
        const uint32_t box[4] = {64, 1, rows, 1};
        const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)heads, (uint64_t)a.S, (uint64_t)a.Z};
        const uint64_t strides[3] = {(uint64_t)a.D * 2, (uint64_t)ld * 2, (uint64_t)a.S * ld * 2};
        return zg::tensor_map_bf16(m, p, 4, dims, strides, box, true);
    };
    if (!map(&tq, a.q, a.H, a.ldq, 128) || !map(&tk, a.k, a.K, a.ldk, W::KEYS) || !map(&tv, a.v, a.K, a.ldv, W::KEYS))
        return zg::fail(ZG_ERR_CUDA, "zg_window_attention: tensor maps");
    if (cudaFuncSetAttribute(window_tc_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W::SMEM) !=
        cudaSuccess)
        return zg::fail(ZG_ERR_CUDA, "zg_window_attention: shared memory attribute");
    const int pairs = (a.S + 255) / 256;
    const int64_t units = (int64_t)a.Z * a.H * pairs;
    if (units > INT32_MAX) return zg::fail(ZG_ERR_INVALID, "zg_window_attention: too many rows");
    zg::LaunchTimer zg_lt_("window_attention", st);
    window_tc_kernel<DP><<<(unsigned)units, WT_THREADS, W::SMEM, st>>>(tq, tk, tv, a, pairs);
    return zg::check_launch("zg_window_attention");
}

}  // namespace

namespace zg {

// Timed-out waits of the tensor-core kernel (codes 101-109, 111-115) or its
// shared memory not 1024-aligned (110); 0 = none.
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
