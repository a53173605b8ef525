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
    // 2^lift is above twice the sequence's length: weights are taken so much
    // smaller, so that no sum of finite values overflows (O / l is the same)
    int lift;
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

// The blocks of keys that a group of rows visits: those that hold sinks, and
// the window's, lo .. last.
struct Blocks {
    int keys, sinks, lo, last;  // keys of a block, blocks that hold sinks
    __device__ __forceinline__ bool has(int b) const { return b <= last && (b >= lo || b < sinks); }
    __device__ __forceinline__ int next(int b) const { return b + 1 < sinks || b + 1 >= lo ? b + 1 : lo; }
};

constexpr int WIN_BAD = 8;  // blocks that are listed by number

// A value that is infinite or NaN reaches the rows that see it and no others,
// but a product of tiles multiplies it with the zero weights of the others
// too.  So where that happened the rows are formed once more with zeros in
// such places, and the outputs that see them are written behind that: NaN
// where a column's visible values hold a NaN or infinities of both signs,
// otherwise the infinity.  On the FMA path that is done here, by one warp, a
// row a lane (`on`: row i takes part: it lies in the sequence, and its weights'
// sum is positive and finite; else all of it is NaN already).  Values are read
// once for the warp's rows; of positions with an infinity also the keys, as a
// weight of exactly zero (a score of -inf) makes it NaN.  blocks[0 .. found -
// 1]: the blocks with such values; more than WIN_BAD: all that the rows visit
// are looked over.  2 x 4096 tokens of 4 heads (2) of 64 in float32, causal,
// 0.51 ms: with one infinite v[0] 0.87, all values NaN 1.2, one column of them
// infinite 5 ms.
template <typename T, int WORDS>
__device__ __noinline__ void window_not_finite(const WindowArgs& a, int z, int h, int i, bool on,
                                               const int* blocks, int found, const Blocks visited) {
    if (!__any_sync(0xffffffffu, on)) return;
    const int lane = threadIdx.x % 32, kh = h / a.G;
    const T* q = static_cast<const T*>(a.q) + ((int64_t)z * a.S + (on ? i : 0)) * a.ldq + (int64_t)h * a.D;
    const T* k = static_cast<const T*>(a.k) + (int64_t)z * a.S * a.ldk + (int64_t)kh * a.D;
    const T* v = static_cast<const T*>(a.v) + (int64_t)z * a.S * a.ldv + (int64_t)kh * a.D;
    const int rows_end = __reduce_max_sync(0xffffffffu, on ? i + 1 : 0);
    uint32_t nan[WORDS], up[WORDS], down[WORDS];  // columns lane' + 32 w of this lane's row as bits
#pragma unroll
    for (int w = 0; w < WORDS; ++w) nan[w] = up[w] = down[w] = 0u;
    constexpr int N = WORDS <= 4 ? 32 / WORDS : 4;  // positions read at a time
    float q_size = -1.f;  // sum of |q|, when it is first needed
    const bool listed = found <= WIN_BAD;
    int at = 0, b = listed ? blocks[0] : visited.sinks > 0 ? 0 : visited.lo;
    while (listed ? at < found : b <= visited.last) {
        const int end = (b + 1) * visited.keys < rows_end ? (b + 1) * visited.keys : rows_end;
        for (int j0 = visited.has(b) ? b * visited.keys : end; j0 < end; j0 += N) {
            T raw[N][WORDS];
#pragma unroll
            for (int g = 0; g < N; ++g)
#pragma unroll
                for (int w = 0; w < WORDS; ++w)
                    raw[g][w] = j0 + g < end && lane + 32 * w < a.D ? v[(j0 + g) * a.ldv + lane + 32 * w] : zg_from_float<T>(0.f);
            float sum = 0.f;  // 0 x is NaN where x is not finite
#pragma unroll
            for (int g = 0; g < N; ++g)
#pragma unroll
                for (int w = 0; w < WORDS; ++w) sum = fmaf(zg_to_float(raw[g][w]), 0.f, sum);
            if (!__any_sync(0xffffffffu, sum != 0.f)) continue;
            uint32_t infinite = 0u;
#pragma unroll
            for (int g = 0; g < N; ++g)
#pragma unroll
                for (int w = 0; w < WORDS; ++w) infinite |= isinf(zg_to_float(raw[g][w])) ? 1u : 0u;
            // whether a weight of these positions may be exactly zero: |q . k| is at most sum |q| max |k|
            bool zeros = false;
            if (__any_sync(0xffffffffu, infinite)) {
                float size = 0.f;
#pragma unroll
                for (int g = 0; g < N; ++g)
#pragma unroll
                    for (int w = 0; w < WORDS; ++w)
                        size = fmaxf(size, fabsf(j0 + g < end && lane + 32 * w < a.D
                                                     ? zg_to_float(k[(j0 + g) * a.ldk + lane + 32 * w]) : 0.f));
#pragma unroll
                for (int f = 16; f > 0; f >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, f));
                if (q_size < 0.f) {
                    q_size = 0.f;
#pragma unroll 16
                    for (int d = 0; d < a.D; ++d) q_size += fabsf(zg_to_float(q[d]));
                }
                zeros = __any_sync(0xffffffffu, on && !(size * q_size < 1e38f));
            }
#pragma unroll
            for (int g = 0; g < N; ++g) {
                const int j = j0 + g;
                const bool see = on && j <= i && j < end && sees(a, i, j);
                bool zero = false;
                if (zeros && j < end) {
                    float score = 0.f;
                    for (int d = 0; d < a.D; ++d) score = fmaf(zg_to_float(q[d]), zg_to_float(k[j * a.ldk + d]), score);
                    zero = score == -INFINITY;
                }
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const float x = zg_to_float(raw[g][w]);
                    const uint32_t bn = __ballot_sync(0xffffffffu, isnan(x)), bu = __ballot_sync(0xffffffffu, x == INFINITY);
                    const uint32_t bd = __ballot_sync(0xffffffffu, x == -INFINITY);
                    if (!see) continue;
                    nan[w] |= zero ? bn | bu | bd : bn;
                    up[w] |= zero ? 0u : bu;
                    down[w] |= zero ? 0u : bd;
                }
            }
        }
        ++at;
        b = !listed ? visited.next(b) : at < found ? blocks[at] : 0;
        bool rest = false;  // a column that may still change
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            const int left = a.D - 32 * w;
            rest = rest || (nan[w] != (left >= 32 ? ~0u : left > 0 ? (1u << left) - 1u : 0u));
        }
        if (!__any_sync(0xffffffffu, on && rest)) break;
    }
    uint32_t any = 0u;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
        nan[w] |= up[w] & down[w];
        any |= nan[w] | up[w] | down[w];
    }
    T* o = static_cast<T*>(a.o) + ((int64_t)z * a.S * a.H + h) * a.D;
    __syncwarp();  // the rows' other columns are written before these
    for (uint32_t rows = __ballot_sync(0xffffffffu, any != 0u); rows; rows &= rows - 1) {
        const int r = __ffs(rows) - 1;
        T* to = o + (int64_t)__shfl_sync(0xffffffffu, i, r) * a.H * a.D;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            const uint32_t rn = __shfl_sync(0xffffffffu, nan[w], r), ru = __shfl_sync(0xffffffffu, up[w], r);
            const uint32_t rd = __shfl_sync(0xffffffffu, down[w], r);
            if ((rn | ru | rd) >> lane & 1)
                to[lane + 32 * w] = zg_from_float<T>(rn >> lane & 1 ? __int_as_float(0x7fffffff)
                                                     : ru >> lane & 1 ? INFINITY : -INFINITY);
        }
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
    const float low = ldexpf(1.f, -a.lift);
    float2 x[4][NC];
    float m[4], l[4];
    const int last = i0 + WF_M < n ? i0 + WF_M : n;  // rows [i0, last)
    const int kt_end = (last + WF_N - 1) / WF_N;
    const int w0 = i0 - a.window + 1 > 0 ? (i0 - a.window + 1) / WF_N : 0;  // the window's first tile
    int sink_end = (a.sinks + WF_N - 1) / WF_N;                              // tiles that hold sinks
    if (sink_end > w0) sink_end = w0;
    auto next = [&](int kt) { return kt + 1 < sink_end || kt >= w0 ? kt + 1 : w0; };
    // Where an output is not finite although the weights' sum is, a value of
    // a visited tile is not: the block goes over its tiles once more, with
    // zeros in such places, and notes the tiles.
    __shared__ int tiles[WIN_BAD];
    int found = 0;
    // (Two instances: with the test in one, 3 x 777 tokens of 8 heads of 80 took 55.0 us instead of 51.3.)
    auto pass = [&](auto second) {
        constexpr bool CLEAN = decltype(second)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) x[i][c] = zero2;
        }
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
                        const float p = exp2f(s[j] - base) * low;
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
            if constexpr (CLEAN) {
                bool bad = false;
                for (int e = threadIdx.x; e < WF_N * DP; e += WF_THREADS) {
                    float& value = vs[e / DP * PITCH + e % DP];
                    if (!isfinite(value)) {
                        value = 0.f;
                        bad = true;
                    }
                }
                if (__syncthreads_or(bad)) {
                    if (threadIdx.x == 0 && found < WIN_BAD) tiles[found] = kt;
                    ++found;
                }
            }
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
        unsigned known = 0;  // bit i: row i's weights have a finite sum (else all of it is NaN, by its visible scores)
        bool fine = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int f = 8; f > 0; f >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], f);
            const int qi = i0 + ty + 8 * i;
            if (l[i] > 0.f && l[i] < INFINITY) known |= 1u << i;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = 32 * c + 2 * tx + e;
                    const float y = qi < n ? (e ? x[i][c].y : x[i][c].x) / l[i] : 0.f;
                    if (d < a.D) {
                        fine = fine && (isfinite(y) || !(known >> i & 1));
                        if (qi < a.S) o[qi * ldo + d] = zg_from_float<T>(y);
                    }
                }
        }
        if constexpr (CLEAN) {
            // lane r: row (r % 2) + 8 (r / 2) of this warp's eight
            const int lane = threadIdx.x % 32, i = i0 + (int)(threadIdx.x / 32) * 2 + lane % 2 + 8 * (lane / 2);
            const unsigned bits = __shfl_sync(0xffffffffu, known, 16 * (lane % 2));
            if (found)
                window_not_finite<T, NC>(a, z, h, i, lane < 8 && i < n && (bits >> (lane / 2 & 3) & 1), tiles, found,
                                         Blocks{WF_N, sink_end, w0, kt_end - 1});
        }
        return fine;
    };
    if (__syncthreads_or(!pass(std::false_type{}))) pass(std::true_type{});
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
// tokens of 16 heads (4) of 128 under a window of 1024: 85 us, 0.76 PFLOP/s.
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
    int w0, lo, last;  // the first position of the unit's window; the first block of this tile's, and its last (-1: a tile behind the sequence)
    bool any, both;  // whether the sequence reaches the first tile, and the second
    __device__ __forceinline__ bool takes(int b) const { return b <= last && (b >= lo || b < sink_blocks); }
    __device__ __forceinline__ int first() const { return sink_blocks > 0 ? 0 : lo0; }
    // whether the blocks that hold sinks hold no other keys that a row sees
    __device__ __forceinline__ bool sinks_apart(int keys) const { return sink_blocks * keys <= w0; }
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
    x.w0 = x.i0 - a.window + 1;
    const int w = x.w0 + 128 * t;
    x.lo0 = x.w0 > 0 ? x.w0 / KEYS : 0;
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

// Whether a value that the blocks of a warp's 32 rows (from row0) hold and
// that not all of them see is not finite: behind the first row, before the
// last one's window, or beside the sinks.
template <int KEYS>
__device__ __forceinline__ bool masked_not_finite(const WindowArgs& a, const WtUnit& x, int row0) {
    const int words = a.D / 8, last = row0 + 31 < x.n - 1 ? row0 + 31 : x.n - 1;
    const int end = (x.last + 1) * KEYS < x.n ? (x.last + 1) * KEYS : x.n;
    const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
    __nv_bfloat162 sum = zero;  // 0 x is NaN where x is not finite
#pragma unroll 1
    for (int part = 0; part < 3; ++part) {
        if (part == 2 && x.sinks_apart(KEYS)) break;
        const int from = part == 0 ? row0 + 1 : part == 1 && x.lo * KEYS > a.sinks ? x.lo * KEYS : a.sinks;
        const int to = part == 0 ? end : part == 1 ? last - a.window + 1 : x.sink_blocks * KEYS < end ? x.sink_blocks * KEYS : end;
        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v) + ((int64_t)x.z * a.S + from) * a.ldv + (int64_t)(x.h / a.G) * a.D;
#pragma unroll 4
        for (int at = threadIdx.x % 32; at < (to - from) * words; at += 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(v + at / words * a.ldv + at % words * 8);
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.x), zero, sum);
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.y), zero, sum);
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.z), zero, sum);
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.w), zero, sum);
        }
    }
    return __any_sync(0xffffffffu, __low2float(sum) != 0.f || __high2float(sum) != 0.f);
}

// Rows r0 .. of the set bits of `rows` once more, by one warp: 16 keys at a
// time as in the paged kernel (a ring of tiles by cp.async, m16n8k16
// products, a running maximum), over what any of the rows sees, with zeros
// for values that are infinite or NaN.  Then those values are written into
// the outputs that see them: of the blocks that held any, products of the mask
// with ones in their places count in each output the visible NaN and
// infinities of either sign.  (A visible score of -inf is a weight of zero,
// and 0 x inf is NaN.)  ring: 24 KB of this warp's.  2 x 4096 tokens of 12
// heads (4) of 64, causal, 0.10 ms a call: with one infinite v[0], which only
// rows that see it meet, the same; with a NaN 60 positions before the end 0.43;
// all values NaN, or one column infinite, 1.9 ms (0.6 us for 16 keys and 16
// rows).
template <int DP>
__device__ __forceinline__ void window_rows(const WindowArgs& a, uint8_t* ring, int z, int h, int n, int r0, uint32_t rows) {
    using T = __nv_bfloat16;
    constexpr int TILE = 16 * DP * 2, STAGES = 24576 / (2 * TILE), CPR = DP / 8, ONE = 0x3f80;
    const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4, kh = h / a.G;
    const T* q = static_cast<const T*>(a.q) + (int64_t)z * a.S * a.ldq + (int64_t)h * a.D;
    const T* k = static_cast<const T*>(a.k) + (int64_t)z * a.S * a.ldk + (int64_t)kh * a.D;
    const T* v = static_cast<const T*>(a.v) + (int64_t)z * a.S * a.ldv + (int64_t)kh * a.D;
    T* o = static_cast<T*>(a.o) + ((int64_t)z * a.S * a.H + h) * a.D;
    const int w0 = r0 - a.window + 1, end = r0 + 15 < n - 1 ? r0 + 15 : n - 1;
    const Blocks blocks{16, (a.sinks + 15) / 16, w0 > 0 ? w0 / 16 : 0, end / 16};
    int bad[WIN_BAD], found = 0;  // blocks with such values

    // body(block, its keys and values in shared memory), for all blocks or for the bad ones alone
    auto walk = [&](bool all, auto body) {
        int at = 0;
        auto first = [&]() { return all ? (blocks.sinks > 0 ? 0 : blocks.lo) : bad[0]; };
        auto fetch = [&](int stage, int b) {
#pragma unroll
            for (int it = 0; it < CPR / 2; ++it) {
                const int x = it * 32 + lane, r = x / CPR, w = x % CPR;
                const bool on = 16 * b + r < n && w * 8 < a.D;
                const uint32_t to = shared_u32(ring + stage * 2 * TILE) + r * (DP * 2) + ((w ^ (r & 7)) * 16);
                copy16(to, on ? k + (int64_t)(16 * b + r) * a.ldk + w * 8 : k, on ? 16 : 0);
                copy16(to + TILE, on ? v + (int64_t)(16 * b + r) * a.ldv + w * 8 : v, on ? 16 : 0);
            }
        };
        auto after = [&](int b, int& i) { return all ? blocks.next(b) : ++i < found ? bad[i] : INT32_MAX; };
        int ahead = first(), ahead_at = 0;
        for (int s = 0; s < STAGES - 1; ++s) {
            if (ahead <= blocks.last) {
                fetch(s, ahead);
                ahead = after(ahead, ahead_at);
            }
            copy_commit();
        }
        int stage = 0;
        for (int b = first(); b <= blocks.last; b = after(b, at)) {
            copy_wait<STAGES - 2>();
            __syncwarp();
            if (ahead <= blocks.last) {
                fetch((stage + STAGES - 1) % STAGES, ahead);
                ahead = after(ahead, ahead_at);
            }
            copy_commit();
            const uint32_t kt = shared_u32(ring + stage * 2 * TILE);
            body(b, kt, kt + TILE);
            stage = (stage + 1) % STAGES;
        }
        copy_wait<0>();
        __syncwarp();
    };

    uint32_t qf[DP / 16][4];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = r0 + g + 8 * (e & 1) < n ? r0 + g + 8 * (e & 1) : n - 1, d = 16 * t + 2 * c + 8 * (e >> 1);
            qf[t][e] = d < a.D ? *reinterpret_cast<const uint32_t*>(q + i * a.ldq + d) : 0u;
        }
    const int k_row = (lane % 8) + 8 * (lane / 16), k_word = (lane / 8) % 2;
    const int v_row = (lane % 8) + 8 * ((lane / 8) % 2), v_word = lane / 16;
    auto scores = [&](float (&s)[2][4], uint32_t kt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = 0.f;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            uint32_t f[4];
            ldmatrix4(f, kt + k_row * (DP * 2) + (((2 * t + k_word) ^ (k_row & 7)) * 16));
            mma_bf16(s[0], qf[t], f[0], f[1]);
            mma_bf16(s[1], qf[t], f[2], f[3]);
        }
    };
    auto values = [&](uint32_t (&f)[4], uint32_t vt, int t) {
        ldmatrix4_t(f, vt + v_row * (DP * 2) + (((2 * t + v_word) ^ (v_row & 7)) * 16));
    };
    // rows r0 + g and r0 + g + 8; a score's or an output's element e is of the row e / 2, and of the
    // key or column 8 j + 2 c + e % 2
    auto sees_key = [&](int b, int j, int e) {
        const int i = r0 + g + 8 * (e >> 1), key = 16 * b + 8 * j + 2 * c + (e & 1);
        return key <= i && sees(a, i, key);
    };
    float l[2] = {0.f, 0.f};
    {
        float x[DP / 8][4], m[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) x[d][0] = x[d][1] = x[d][2] = x[d][3] = 0.f;
        const float low = ldexpf(1.f, -a.lift);
        walk(true, [&](int b, uint32_t kt, uint32_t vt) {
            float s[2][4];
            scores(s, kt);
            float top[2] = {m[0], m[1]}, f[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[j][e] = sees_key(b, j, e) ? s[j][e] * a.scale : -INFINITY;
                    top[e >> 1] = fmaxf(top[e >> 1], s[j][e]);
                }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                const float base = top[r] == -INFINITY ? 0.f : top[r];
                f[r] = exp2_fast(m[r] - base);
                m[r] = top[r];
                l[r] *= f[r];
                top[r] = base;
            }
#pragma unroll
            for (int d = 0; d < DP / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[d][e] *= f[e >> 1];
            uint32_t p[4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float y0 = exp2_fast(s[j][2 * r] - top[r]) * low, y1 = exp2_fast(s[j][2 * r + 1] - top[r]) * low;
                    l[r] += y0 + y1;
                    p[2 * j + r] = pack_bf16(y0, y1);
                }
            bool spoilt = false;
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
                uint32_t w[4];
                values(w, vt, t);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool lo = (w[e] & 0x7f80u) == 0x7f80u, hi = (w[e] & 0x7f800000u) == 0x7f800000u;
                    spoilt = spoilt || lo || hi;
                    w[e] &= (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
                }
                mma_bf16(x[2 * t], p, w[0], w[1]);
                mma_bf16(x[2 * t + 1], p, w[2], w[3]);
            }
            if (__any_sync(0xffffffffu, spoilt)) {
                if (found < WIN_BAD) bad[found] = b;
                ++found;
            }
        });
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (!(rows >> (g + 8 * r) & 1)) continue;
#pragma unroll
            for (int d = 0; d < DP / 8; ++d)
                if (8 * d < a.D)
                    *reinterpret_cast<uint32_t*>(o + (int64_t)(r0 + g + 8 * r) * a.H * a.D + 8 * d + 2 * c) =
                        pack_bf16(x[d][2 * r] / l[r], x[d][2 * r + 1] / l[r]);
        }
    }
    if (!found) return;
    float up[DP / 8][4], down[DP / 8][4];  // visible +inf or NaN, and -inf or NaN
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) up[d][e] = down[d][e] = 0.f;
    walk(found > WIN_BAD, [&](int b, uint32_t kt, uint32_t vt) {
        float s[2][4];
        scores(s, kt);
        uint32_t some[4], none[4];  // ones where the weight is above zero, and where it is zero
        bool zeros = false;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                some[2 * j + r] = none[2 * j + r] = 0u;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (!sees_key(b, j, 2 * r + e)) continue;
                    const bool zero = s[j][2 * r + e] == -INFINITY;
                    (zero ? none : some)[2 * j + r] |= ONE << 16 * e;
                    zeros = zeros || zero;
                }
            }
        zeros = __any_sync(0xffffffffu, zeros);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            uint32_t w[4], wu[4], wd[4];
            values(w, vt, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                wu[e] = wd[e] = 0u;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t y = w[e] >> 16 * x & 0xffffu;
                    if ((y & 0x7fffu) > 0x7f80u || y == 0x7f80u) wu[e] |= ONE << 16 * x;
                    if ((y & 0x7fffu) > 0x7f80u || y == 0xff80u) wd[e] |= ONE << 16 * x;
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mma_bf16(up[2 * t + e], some, wu[2 * e], wu[2 * e + 1]);
                mma_bf16(down[2 * t + e], some, wd[2 * e], wd[2 * e + 1]);
            }
            if (!zeros) continue;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mma_bf16(up[2 * t + e], none, wu[2 * e] | wd[2 * e], wu[2 * e + 1] | wd[2 * e + 1]);
                mma_bf16(down[2 * t + e], none, wu[2 * e] | wd[2 * e], wu[2 * e + 1] | wd[2 * e + 1]);
            }
        }
    });
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = e >> 1;
            const bool known = l[r] > 0.f && l[r] < INFINITY;  // else all of the row is NaN
            if (8 * d < a.D && known && (rows >> (g + 8 * r) & 1) && (up[d][e] > 0.f || down[d][e] > 0.f))
                o[(int64_t)(r0 + g + 8 * r) * a.H * a.D + 8 * d + 2 * c + (e & 1)] =
                    __float2bfloat16(up[d][e] > 0.f && down[d][e] > 0.f ? __int_as_float(0x7fffffff)
                                     : up[d][e] > 0.f ? INFINITY : -INFINITY);
        }
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
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmSinks, const WindowArgs a,
                 int pairs) {
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
                        // the values beside the sinks, that nobody sees, as zeros (they may be infinite or NaN)
                        tma_load_4d(to + W::BLOCK, b < x.sink_blocks && x.sinks_apart(W::KEYS) ? &tmSinks : &tmV,
                                    &c.kv_full[st], 64 * d, kh, b * W::KEYS, x.z);
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
        const float lift = (float)a.lift + 8.f, slack = 8.f - lift;  // weights up to 2^8 times those of the maximum
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
            float m = -INFINITY;  // what the weights are taken against, in units of log2: a maximum so far, and lift
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            bool first = true;
            for (int b = x.first(); b <= x.hi; b = x.next(b)) {
                if (!x.takes(b)) continue;
                const uint32_t sc = trow + W::s_col(t), pc = trow + W::p_col(t, nb);
                if (!s_ready && !(ok = warp_wait(&c.s_full[t], nb & 1, 111))) break;
                tc_fence_after();
                const int j0 = b * W::KEYS;
                // m is moved to the row's maximum (mx, scaled) and lift where that is
                // more than 2^8 above the one it was taken from; false when a wait ran out.
                auto settle = [&](float mx, bool pv_seen) {
                    // P V of the block before has read the weights' buffer and added to O
                    const bool all_seen = __all_sync(0xffffffffu, pv_seen);
                    if (W::PB == 1 && !first) {
                        if (!all_seen && !warp_wait(&c.pv_done[t], (nb - 1) & 1, 112)) return false;
                        tc_fence_after();
                    }
                    if (!__any_sync(0xffffffffu, i < x.n && !(mx <= m + slack))) return true;  // rows behind the sequence do not count
                    const float n = fmaxf(m, mx + lift);
                    float f = exp2_fast(m - (n == -INFINITY ? 0.f : n));
                    // a score that is NaN or +inf makes the weights' sum NaN, and with it all of the row
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
            const bool again = in && !fine && l > 0.f && l < INFINITY;
            if (__any_sync(0xffffffffu, again) && masked_not_finite<W::KEYS>(a, x, row0)) {
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
        const int last = ok ? c.redo[warp - 4] : -1;
        tc_fence_before();
        __syncthreads();
        // The marked rows, the last unit's first, when nobody waits for this warp
        // and the ring of blocks is free.
        for (int u = last; u >= 0;) {
            const WtUnit x = wt_unit<W::KEYS>(a, u, pairs, t);
            const int row0 = x.i0 + 128 * t + 32 * quad, i = row0 + lane;
            const __nv_bfloat16* o = static_cast<const __nv_bfloat16*>(a.o) + ((int64_t)x.z * a.S + i) * ldo + (int64_t)x.h * a.D;
            const bool again = i < x.n && *reinterpret_cast<const volatile uint16_t*>(o) == WT_REDO;
            const int before = again ? *reinterpret_cast<const volatile int*>(o + 2) : -1;
            const uint32_t rows = __ballot_sync(0xffffffffu, again);
            u = __shfl_sync(0xffffffffu, before, __ffs(rows) - 1);
#pragma unroll 1
            for (int half = 0; half < 2; ++half)
                if (rows >> 16 * half & 0xffffu)
                    window_rows<DP>(a, smem + (warp - 4) * 24576, x.z, x.h, x.n, row0 + 16 * half, rows >> 16 * half & 0xffffu);
        }
        return;
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
    CUtensorMap tq, tk, tv, ts;
    auto map = [&](CUtensorMap* m, const void* p, int heads, int64_t ld, uint32_t rows, int positions) {
        const uint32_t box[4] = {64, 1, rows, 1};
        const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)heads, (uint64_t)positions, (uint64_t)a.Z};
        const uint64_t strides[3] = {(uint64_t)a.D * 2, (uint64_t)ld * 2, (uint64_t)a.S * ld * 2};
        return zg::tensor_map_bf16(m, p, 4, dims, strides, box, true);
    };
    if (!map(&tq, a.q, a.H, a.ldq, 128, a.S) || !map(&tk, a.k, a.K, a.ldk, W::KEYS, a.S) ||
        !map(&tv, a.v, a.K, a.ldv, W::KEYS, a.S) || !map(&ts, a.v, a.K, a.ldv, W::KEYS, a.sinks > 0 ? a.sinks : 1))
        return zg::fail(ZG_ERR_CUDA, "zg_window_attention: tensor maps");
    if (cudaFuncSetAttribute(window_tc_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W::SMEM) !=
        cudaSuccess)
        return zg::fail(ZG_ERR_CUDA, "zg_window_attention: shared memory attribute");
    const int pairs = (a.S + 255) / 256;
    const int64_t units = (int64_t)a.Z * a.H * pairs;
    if (units > INT32_MAX) return zg::fail(ZG_ERR_INVALID, "zg_window_attention: too many rows");
    zg::LaunchTimer zg_lt_("window_attention", st);
    window_tc_kernel<DP><<<(unsigned)units, WT_THREADS, W::SMEM, st>>>(tq, tk, tv, ts, a, pairs);
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
    if (Z < 0 || S < 0 || Z > INT32_MAX || S > (1 << 30) || H < 1 || K < 1 || H % K || D < 1 || Z > INT32_MAX / H)
        return zg::fail(ZG_ERR_INVALID, "zg_window_attention: bad sizes");
    if (D > 256) return zg::fail(ZG_ERR_UNSUPPORTED, "zg_window_attention: head dim above 256");
    if (window < 0 || sinks < 0)
        return zg::fail(ZG_ERR_INVALID, "zg_window_attention: window and sinks must be >= 0");
    if (ldq < (int64_t)H * D || ldk < (int64_t)K * D || ldv < (int64_t)K * D)
        return zg::fail(ZG_ERR_INVALID, "zg_window_attention: row pitch below heads * D");
    if (!zg::dtype_ok(dtype)) return zg::fail(ZG_ERR_INVALID, "zg_window_attention: bad dtype");
    if (Z == 0 || S == 0) return ZG_OK;
    if (!q || !k || !v || !o) return zg::fail(ZG_ERR_INVALID, "zg_window_attention: null pointer");
    int lift = 1;
    while (((int64_t)1 << (lift - 1)) <= S) ++lift;
    const WindowArgs a{q, k, v, o, lengths, ldq, ldk, ldv, (int)Z, (int)S, H, K, D, H / K,
                       window > 0 && window < S ? window : (int)S, sinks < S ? sinks : (int)S,
                       (float)(1.4426950408889634 / sqrt((double)D)), lift};
    cudaStream_t st = zg::as_stream(stream);
    auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if (dtype == ZG_BF16 && D <= 128 && D % 8 == 0 && ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && al(q) && al(k) &&
        al(v) && al(o) && zg::tc_available())
        return D <= 64 ? launch_window_tc<64>(a, st) : launch_window_tc<128>(a, st);
    return dtype == ZG_BF16 ? launch_window_any<__nv_bfloat16>(a, st) : launch_window_any<float>(a, st);
}
