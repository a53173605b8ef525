// zg_rotary.cu -- rotary positions with one or several axes, applied to the
// queries and the keys of a candidate's attention in one launch.
//
//   pair p of a head (columns a, b), of axis x_p and frequency f_p:
//     t   = position[token, x_p] * f_p
//     y_a = x_a cos t - x_b sin t,   y_b = x_a sin t + x_b cos t
//   f_p = base^(-e_p); e_p counts the pairs of the axis (or, joint, of all
//   axes) in [0, 1).  inverse turns by -t (the transpose).
//
// HBM-bound: every element is read once and written once.  The angles are
// the only arithmetic that is not a few FMAs per element, so a block takes
// a few tokens, puts their (cos, sin) in shared memory once and turns all
// the heads of q and k with them (16 to 40 heads share an angle).  An angle
// is formed in turns, position * f / (2 pi), in 64 bits and reduced to its
// nearest turn there (a position of 10^6 loses 0.06 rad in float32); only
// the reduced angle goes to sincospif.
#include <math.h>

#include "zg_ptx.cuh"

namespace {

constexpr int RO_MAX_PAIRS = 128;  // D <= 256
constexpr int RO_THREADS = 128;

enum { RO_POS_I32 = 0, RO_POS_I64 = 1, RO_POS_F32 = 2 };

// Division of x by d as a product with ceil(2^32 / d): exact while x d < 2^32.
struct Div {
    uint32_t magic, one;  // one: all bits where d = 1
    __device__ __forceinline__ int operator()(int x) const { return (int)(__umulhi((uint32_t)x, magic) + ((uint32_t)x & one)); }
};
Div divide_by(int64_t d) { return d == 1 ? Div{0u, ~0u} : Div{(uint32_t)(((1ull << 32) + d - 1) / d), 0u}; }

struct RotaryArgs {
    const void *q, *k, *pos;
    void *q_out, *k_out;
    int64_t ldq, ldk, T, pos_rows;
    int H, K, D, A, pairs, pos_type, interleaved, tokens;  // tokens: per block
    float sign;
    Div by_pairs, by_token, by_head;  // items of a token (0 for a token a block), and of a head
    double turns[RO_MAX_PAIRS];  // f_p / (2 pi)
    uint8_t axis[RO_MAX_PAIRS];
};

// (cos, sin) of every pair p of the block's nt tokens from t0, handed to
// put(token, p, cos, sin).  The row of a position table that repeats is found
// once a block (a 64-bit remainder costs some hundred instructions).
template <typename F>
__device__ __forceinline__ void rotary_angles(const RotaryArgs& a, int64_t t0, int nt, F put) {
    const int64_t row0 = t0 % a.pos_rows;
    for (int i = threadIdx.x; i < nt * a.pairs; i += RO_THREADS) {
        const int tt = a.by_pairs(i), p = i - tt * a.pairs;
        int64_t row = row0 + tt;
        while (row >= a.pos_rows) row -= a.pos_rows;
        const int64_t at = row * a.A + a.axis[p];
        const double x = a.pos_type == RO_POS_I64   ? (double)static_cast<const int64_t*>(a.pos)[at]
                         : a.pos_type == RO_POS_I32 ? (double)static_cast<const int32_t*>(a.pos)[at]
                                                    : (double)static_cast<const float*>(a.pos)[at];
        const double t = x * a.turns[p];
        float s, c;
        sincospif((float)(2.0 * (t - rint(t))), &s, &c);
        put(tt, p, c, s * a.sign);
    }
}

// Sixteen bytes of T as floats, and back.
template <typename T>
struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[N]) {
        if constexpr (sizeof(T) == 2) {
            bf16x8_to_f32(r, v);
        } else {
            v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y);
            v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[N]) {
        uint4 r;
        if constexpr (sizeof(T) == 2) {
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        } else {
            r = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        }
        return r;
    }
};

// Rows of 16-byte words.  An item is one word of an interleaved head, or two
// words (the pairs' two columns) of a head in halves; the unturned columns
// behind the pairs are items of one word, copied.  A thread has RO_ITEMS
// items' words on the way at a time, the first ones while the block forms its
// angles.  336 MB of bf16 (two videos of 16384 tokens, 16 + 4 heads of 128):
// 64 us, 5.3 TB/s (66 with an item's token and head by the compiler's integer
// divisions); with the angles read one by one, lanes 64 bytes apart in
// shared memory, 74 us (the reads of four lanes met in a bank); persistent
// blocks that fetch a group of tokens ahead by cp.async, 84 us (an SM's
// instructions, not its reads in flight, are what is left).
constexpr int RO_ITEMS = 4;

template <typename T, bool IL>
__global__ void __launch_bounds__(RO_THREADS) rotary_vec_kernel(const __grid_constant__ RotaryArgs a) {
    constexpr int N = Vec16<T>::N;
    // An item's angles two by two, (cos, cos, sin, sin), those of neighbouring
    // items of a head side by side: [tokens][EACH / 2][turned], EACH its pairs.
    constexpr int EACH = IL ? N / 2 : N;
    extern __shared__ float4 table[];
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
    const int nt = (int)(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
    const int turned = IL ? 2 * a.pairs / N : a.pairs / N;  // items of a head that are turned
    const int per_head = turned + (a.D - 2 * a.pairs) / N;
    const int per_token = per_head * (a.H + a.K);
    bool angles = false;
    for (int i0 = 0; i0 < nt * per_token; i0 += RO_ITEMS * RO_THREADS) {
        uint4 u[RO_ITEMS], z[IL ? 1 : RO_ITEMS];
        int tt[RO_ITEMS], col[RO_ITEMS];  // token of the block, first column; col < 0: no item
        T* y[RO_ITEMS];
#pragma unroll
        for (int e = 0; e < RO_ITEMS; ++e) {
            const int i = i0 + e * RO_THREADS + threadIdx.x;
            col[e] = -1;
            if (i >= nt * per_token) continue;
            tt[e] = a.by_token(i);
            const int r = i - tt[e] * per_token, hh = a.by_head(r), c = r - hh * per_head;
            const int64_t token = t0 + tt[e];
            const bool is_q = hh < a.H;
            const int h = is_q ? hh : hh - a.H;
            const T* x = static_cast<const T*>(is_q ? a.q : a.k) + token * (is_q ? a.ldq : a.ldk) + (int64_t)h * a.D;
            y[e] = static_cast<T*>(is_q ? a.q_out : a.k_out) + (token * (is_q ? a.H : a.K) + h) * a.D;
            col[e] = c < turned ? c * N : 2 * a.pairs + (c - turned) * N;
            u[e] = *reinterpret_cast<const uint4*>(x + col[e]);
            if constexpr (!IL)
                if (c < turned) z[e] = *reinterpret_cast<const uint4*>(x + a.pairs + col[e]);
        }
        if (!angles) {
            rotary_angles(a, t0, nt, [&](int token, int p, float cosine, float sine) {
                float* at = reinterpret_cast<float*>(table + (token * (EACH / 2) + p % EACH / 2) * turned + p / EACH);
                at[p & 1] = cosine;
                at[2 + (p & 1)] = sine;
            });
            __syncthreads();
            angles = true;
        }
#pragma unroll
        for (int e = 0; e < RO_ITEMS; ++e) {
            if (col[e] < 0) continue;
            if (col[e] >= (IL ? 2 * a.pairs : a.pairs)) {
                *reinterpret_cast<uint4*>(y[e] + col[e]) = u[e];
                continue;
            }
            const float4* w = table + tt[e] * (EACH / 2) * turned + col[e] / N;
            float p[N], s[N];
            Vec16<T>::unpack(u[e], p);
            if constexpr (!IL) Vec16<T>::unpack(z[e], s);
#pragma unroll
            for (int f = 0; f < EACH; f += 2) {
                const float4 g = w[f / 2 * turned];
                const float2 c = make_float2(g.x, g.y), d = make_float2(g.z, g.w), zero = make_float2(0.f, 0.f);
                const float2 o = IL ? make_float2(p[2 * f], p[2 * f + 2]) : make_float2(p[f], p[f + 1]);
                const float2 t = IL ? make_float2(p[2 * f + 1], p[2 * f + 3]) : make_float2(s[f], s[f + 1]);
                const float2 td = ffma2_tc(t, d, zero);
                const float2 ra = ffma2_tc(o, c, make_float2(-td.x, -td.y)), rb = ffma2_tc(o, d, ffma2_tc(t, c, zero));
                if constexpr (IL) {
                    p[2 * f] = ra.x; p[2 * f + 2] = ra.y; p[2 * f + 1] = rb.x; p[2 * f + 3] = rb.y;
                } else {
                    p[f] = ra.x; p[f + 1] = ra.y; s[f] = rb.x; s[f + 1] = rb.y;
                }
            }
            *reinterpret_cast<uint4*>(y[e] + col[e]) = Vec16<T>::pack(p);
            if constexpr (!IL) *reinterpret_cast<uint4*>(y[e] + a.pairs + col[e]) = Vec16<T>::pack(s);
        }
    }
}

// Any width and alignment: an item is one pair, or one unturned column.
template <typename T>
__global__ void __launch_bounds__(RO_THREADS) rotary_any_kernel(const __grid_constant__ RotaryArgs a) {
    extern __shared__ float2 cs[];
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
    const int nt = (int)(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
    rotary_angles(a, t0, nt, [&](int token, int p, float c, float s) { cs[token * a.pairs + p] = make_float2(c, s); });
    __syncthreads();
    const int per_head = a.D - a.pairs, per_token = per_head * (a.H + a.K);
    for (int i = threadIdx.x; i < nt * per_token; i += RO_THREADS) {
        const int tt = i / per_token, r = i - tt * per_token;
        const int hh = r / per_head, c = r - hh * per_head;
        const int64_t token = t0 + tt;
        const bool is_q = hh < a.H;
        const int h = is_q ? hh : hh - a.H;
        const T* x = static_cast<const T*>(is_q ? a.q : a.k) + token * (is_q ? a.ldq : a.ldk) + (int64_t)h * a.D;
        T* y = static_cast<T*>(is_q ? a.q_out : a.k_out) + (token * (is_q ? a.H : a.K) + h) * a.D;
        if (c >= a.pairs) {
            y[c + a.pairs] = x[c + a.pairs];
            continue;
        }
        const float2 f = cs[tt * a.pairs + c];
        const int ca = a.interleaved ? 2 * c : c, cb = a.interleaved ? 2 * c + 1 : c + a.pairs;
        const float u = zg_to_float(x[ca]), z = zg_to_float(x[cb]);
        y[ca] = zg_from_float<T>(u * f.x - z * f.y);
        y[cb] = zg_from_float<T>(u * f.y + z * f.x);
    }
}

template <typename T>
int launch_rotary(RotaryArgs& a, cudaStream_t st) {
    constexpr int N = Vec16<T>::N;
    auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool vec = a.D % N == 0 && (a.interleaved ? 2 * a.pairs : a.pairs) % N == 0 && a.ldq % N == 0 &&
                     a.ldk % N == 0 && al(a.q) && al(a.k) && al(a.q_out) && al(a.k_out);
    // as many tokens a block as its threads have items in flight, fewer while
    // the grid is short of two blocks per SM
    const int pairs_of = a.interleaved ? 2 * a.pairs / N : a.pairs / N;
    const int per_head = vec ? pairs_of + (a.D - 2 * a.pairs) / N : a.D - a.pairs;
    const int64_t items = (int64_t)per_head * (a.H + a.K);
    a.tokens = (int)(RO_ITEMS * RO_THREADS / items);
    if (a.tokens > 16) a.tokens = 16;
    if (a.tokens < 1) a.tokens = 1;
    while (a.tokens > 1 && (a.T + a.tokens - 1) / a.tokens < 2 * 148) a.tokens /= 2;
    // two tokens or more have 512 items at most, and items of a token 2^23
    a.by_pairs = divide_by(a.pairs);
    a.by_token = a.tokens > 1 ? divide_by(items) : Div{0u, 0u};
    a.by_head = divide_by(per_head);
    const int64_t blocks = (a.T + a.tokens - 1) / a.tokens;
    if (blocks > INT32_MAX) return zg::fail(ZG_ERR_INVALID, "zg_rotary: too many tokens");
    const size_t smem = (size_t)a.tokens * a.pairs * sizeof(float2);
    zg::LaunchTimer zg_lt_("rotary", st);
    if (!vec)
        rotary_any_kernel<T><<<(unsigned)blocks, RO_THREADS, smem, st>>>(a);
    else if (a.interleaved)
        rotary_vec_kernel<T, true><<<(unsigned)blocks, RO_THREADS, smem, st>>>(a);
    else
        rotary_vec_kernel<T, false><<<(unsigned)blocks, RO_THREADS, smem, st>>>(a);
    return zg::check_launch("zg_rotary");
}

}  // namespace

extern "C" int zg_rotary(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* positions, int pos_type,
                         int64_t T, int64_t pos_rows, int H, int K, int D, int A, const int32_t* axes, double base,
                         int interleaved, int joint, int inverse, int dtype, void* q_out, void* k_out, void* stream) {
    if (T < 0 || H < 0 || K < 0 || H + (int64_t)K < 1 || H > 65536 || K > 65536 || D < 2 || A < 1 || A > RO_MAX_PAIRS)
        return zg::fail(ZG_ERR_INVALID, "zg_rotary: bad sizes");
    if (D > 2 * RO_MAX_PAIRS) return zg::fail(ZG_ERR_UNSUPPORTED, "zg_rotary: head dim above 256");
    if (ldq < (int64_t)H * D || ldk < (int64_t)K * D)
        return zg::fail(ZG_ERR_INVALID, "zg_rotary: row pitch below heads * D");
    if (!zg::dtype_ok(dtype)) return zg::fail(ZG_ERR_INVALID, "zg_rotary: bad dtype");
    if (pos_type < RO_POS_I32 || pos_type > RO_POS_F32) return zg::fail(ZG_ERR_INVALID, "zg_rotary: bad position type");
    if (!(base > 0.0) || !isfinite(base)) return zg::fail(ZG_ERR_INVALID, "zg_rotary: base must be positive");
    if (!axes) return zg::fail(ZG_ERR_INVALID, "zg_rotary: null pointer");
    RotaryArgs a{};
    int64_t width = 0;
    for (int i = 0; i < A; ++i) {
        if (axes[i] < 2 || axes[i] % 2) return zg::fail(ZG_ERR_INVALID, "zg_rotary: axis widths are even and positive");
        width += axes[i];
    }
    if (width > D) return zg::fail(ZG_ERR_INVALID, "zg_rotary: the axes are wider than the head");
    if (T == 0) return ZG_OK;
    if (pos_rows < 1 || T % pos_rows) return zg::fail(ZG_ERR_INVALID, "zg_rotary: positions do not divide the tokens");
    if (!positions || (H && (!q || !q_out)) || (K && (!k || !k_out)))
        return zg::fail(ZG_ERR_INVALID, "zg_rotary: null pointer");
    a.pairs = (int)(width / 2);
    // base^(-j/n) by repeated products in the host's 64-bit mantissas: at most
    // 127 roundings of 2^-64, below one of the doubles they end in
    const long double start = 1.0L / 6.283185307179586476925286766559005768L;
    long double f = start, step = powl((long double)base, -1.0L / a.pairs);
    for (int i = 0, p = 0; i < A; ++i) {
        if (!joint) {
            f = start;
            step = powl((long double)base, -2.0L / axes[i]);
        }
        for (int j = 0; j < axes[i] / 2; ++j, ++p, f *= step) {
            a.turns[p] = (double)f;
            a.axis[p] = (uint8_t)i;
        }
    }
    a.q = q; a.k = k; a.pos = positions; a.q_out = q_out; a.k_out = k_out;
    a.ldq = ldq; a.ldk = ldk; a.T = T; a.pos_rows = pos_rows;
    a.H = H; a.K = K; a.D = D; a.A = A; a.pos_type = pos_type; a.interleaved = interleaved != 0;
    a.sign = inverse ? -1.f : 1.f;
    cudaStream_t st = zg::as_stream(stream);
    return dtype == ZG_BF16 ? launch_rotary<__nv_bfloat16>(a, st) : launch_rotary<float>(a, st);
}
