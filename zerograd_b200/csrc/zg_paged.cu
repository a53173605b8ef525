// zg_paged.cu -- a paged key-value cache: writing new tokens into its pages,
// and the attention of one new token over them.
//
// Pages are [N, page, K, D] (keys and values apart); a sequence's tokens
// 0 .. length - 1 lie in the pages its row of the page table names, in order.
//
//   append:    token (b, s) of sequence b goes to position lengths[b] + s.
//   attention: o[b, h] = sum_j softmax_j(q[b, h] . k_j / sqrt(D)) v_j over the
//              positions j that the newest token (position length - 1) sees:
//              the last `window` ones and the first `sinks`.
//
// Both are bound by HBM: append moves each token once, and attention reads
// each visible key and value once for the G = H / K query heads that share
// them (4 G D flops on 4 D bytes at bf16: G flops per byte, far below the
// tensor cores' or, in float32, the FMA pipe's rate for any usual G).
#include <math.h>

#include "zg_common.cuh"
#include "zg_warp.cuh"

namespace {

constexpr int PG_WARPS = 4;
constexpr int64_t PG_MOST = 1 << 30;  // positions of a table's row, and of a pool

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendArgs {
    void *kp, *vp;
    const void *k, *v;
    const int32_t *table, *lengths, *counts;
    int32_t* new_lengths;
    int64_t n_pages, ldk, ldv, row;  // row: words (or elements) of a token's K heads
    int64_t rows;                    // B * S
    int page, max_pages, B, S;
};

// The tokens of sequence b that are written: none when they do not fit.
__device__ __forceinline__ bool append_span(const AppendArgs& a, int b, int& start, int& count) {
    start = a.lengths[b];
    count = a.counts ? a.counts[b] : a.S;
    return start >= 0 && count >= 0 && count <= a.S &&
           (int64_t)start + count <= (int64_t)a.max_pages * a.page;
}

// A warp per token, W the word that it is copied in (16 bytes, or one
// element where a row's length or alignment does not allow that), key and
// value words loaded before either is stored, the first ones beside the page
// table's entry.  The warps behind the tokens' own take a sequence each and
// write its new length.
template <typename W>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x % 32;
    const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
    int start, count;
    if (w >= a.rows) {
        const int64_t b = w - a.rows;
        if (b >= a.B) return;
        bool ok = append_span(a, (int)b, start, count);
        if (ok && count > 0) {
            const int last = (start + count - 1) / a.page;
            bool bad = false;
            for (int p = start / a.page + lane; p <= last; p += 32) {
                const int32_t id = a.table[b * a.max_pages + p];
                bad |= id < 0 || id >= a.n_pages;
            }
            ok = !__any_sync(0xffffffffu, bad);
        }
        if (lane == 0) a.new_lengths[b] = ok ? start + count : -1;
        return;
    }
    // (a 64-bit quotient costs some hundred instructions)
    const int b = w <= INT32_MAX ? (int)((uint32_t)w / (uint32_t)a.S) : (int)(w / a.S), s = (int)(w - (int64_t)b * a.S);
    if (!append_span(a, b, start, count) || s >= count) return;
    const int at = start + s, p = at / a.page;
    const W* ks = static_cast<const W*>(a.k) + w * a.ldk;
    const W* vs = static_cast<const W*>(a.v) + w * a.ldv;
    const int32_t id = a.table[(int64_t)b * a.max_pages + p];
    W k0{}, k1{}, v0{}, v1{};
    auto take = [&](int64_t i) {
        if (i < a.row) k0 = ks[i], v0 = vs[i];
        if (i + 32 < a.row) k1 = ks[i + 32], v1 = vs[i + 32];
    };
    take(lane);
    if (id < 0 || id >= a.n_pages) return;
    const int64_t to = ((int64_t)id * a.page + (at - p * a.page)) * a.row;
    W* kd = static_cast<W*>(a.kp) + to;
    W* vd = static_cast<W*>(a.vp) + to;
    for (int64_t i = lane; i < a.row;) {
        kd[i] = k0;
        vd[i] = v0;
        if (i + 32 < a.row) {
            kd[i + 32] = k1;
            vd[i + 32] = v1;
        }
        i += 64;
        take(i);
    }
}

// ---------------------------------------------------------------------------
// attention of one token
// ---------------------------------------------------------------------------
struct PagedArgs {
    const void *q, *kp, *vp;
    const int32_t *table, *lengths;
    void* o;
    float* part;  // share > 0: of each block m [R], l [R], then R rows of sums
    int64_t ldq, n_pages;
    int page, max_pages, B, H, K, D, G, row_tiles, R;  // R: query rows of a unit (heads that share a key head)
    // splits > 1: a unit's splits are a cluster, which joins them; share > 0:
    // so many blocks have equal shares of all units, joined by a kernel
    int window, sinks, splits, share;
    float scale;  // log2(e) / sqrt(D)
};

__host__ __device__ __forceinline__ int pad4(int d) { return (d + 3) / 4 * 4; }
__host__ __device__ __forceinline__ int64_t part_floats(int R, int D) { return 2 * (int64_t)R + (int64_t)R * pad4(D); }

// What the newest of `length` tokens sees: positions 0 .. s-1 and, behind a
// gap, the last of them; vis of them in all.  vis < 0: the length is not one
// the table can hold.
struct Seen {
    int vis, s, gap;
    __device__ __forceinline__ int token(int t) const { return t < s ? t : t + gap; }
};
__device__ __forceinline__ Seen seen_by(const PagedArgs& a, int b) {
    const int n = a.lengths[b];
    if (n < 0 || (int64_t)n > (int64_t)a.max_pages * a.page) return Seen{-1, 0, 0};
    const int w = a.window > 0 && a.window < n ? a.window : n;
    const int s = a.sinks < n - w ? a.sinks : n - w;
    return Seen{w + s, s, n - w - s};
}

constexpr int PG_MIN_CHUNK = 128;  // positions of a share: less would be the pipeline's filling and the join

// The blocks' equal shares, from the sequences' lengths (at most 64 of them):
// lane l has those of sequences 2 l and 2 l + 1.
struct Shares {
    int chunk, splits[2], before;  // positions of a share, shares of one unit, blocks of the sequences before 2 l
};
__device__ __forceinline__ Shares shares_of(const PagedArgs& a) {
    const int lane = threadIdx.x % 32, heads = a.K * a.row_tiles;
    if (a.B == 1) {
        const int v = lane == 0 ? seen_by(a, 0).vis : 0, each = a.share / heads;
        const int even = ((v < 0 ? 0 : v) + each - 1) / each;
        const int chunk = __shfl_sync(0xffffffffu, ((even < PG_MIN_CHUNK ? PG_MIN_CHUNK : even) + 63) / 64 * 64, 0);
        return Shares{chunk, {v > 0 ? (v + chunk - 1) / chunk : 0, 0}, 0};
    }
    int vis[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        vis[j] = 2 * lane + j < a.B ? seen_by(a, 2 * lane + j).vis : 0;
        if (vis[j] < 0) vis[j] = 0;
    }
    long long total = (long long)vis[0] + vis[1];
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    // the shortest shares that there are blocks for: from those that would all
    // be full, a quarter of the way at a time, to those that are enough even if
    // each unit ends in a share of its own
    auto part = [&](int blocks) {
        const int even = (int)ceil((double)(total * heads) / blocks);  // exact below 2^53
        return ((even < PG_MIN_CHUNK ? PG_MIN_CHUNK : even) + 63) / 64 * 64;
    };
    const int least = part(a.share), most = part(a.share - a.B * heads);
    Shares h;
    h.chunk = most;
#pragma unroll 1
    for (int k = 0; k < 4 && least < most; ++k) {
        const int c = least + (most - least) / 64 * k / 4 * 64;
        int used = heads * ((vis[0] + c - 1) / c + (vis[1] + c - 1) / c);
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) used += __shfl_xor_sync(0xffffffffu, used, x);
        if (used <= a.share) {
            h.chunk = c;
            break;
        }
    }
    int n = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        h.splits[j] = (vis[j] + h.chunk - 1) / h.chunk;
        n += heads * h.splits[j];
    }
    h.before = n;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, h.before, x);
        if ((int)threadIdx.x % 32 >= x) h.before += below;
    }
    h.before -= n;
    return h;
}

// What this block does: positions c0 .. c0 + chunk - 1 of what row tile rt of
// key head kh of sequence b sees.  on: it has any share.
struct Work {
    int b, kh, rt, split, c0, chunk;
    bool on;
};
// (SHARE, a.share > 0, is an instance of its own: with both in one, 64
// sequences took 80.1 us instead of 77.9.)
template <bool SHARE>
__device__ __forceinline__ Work work_of(const PagedArgs& a) {
    Work w;
    int unit;
    w.on = true;
    if constexpr (SHARE) {
        const int lane = threadIdx.x % 32, x = (int)blockIdx.x, heads = a.K * a.row_tiles;
        const Shares h = shares_of(a);
        const int mine = heads * (h.splits[0] + h.splits[1]);
        const unsigned at = __ballot_sync(0xffffffffu, x >= h.before && x < h.before + mine);
        w.on = at != 0;
        const int from = w.on ? __ffs(at) - 1 : 0;
        int left = x - __shfl_sync(0xffffffffu, h.before, from);
        int splits = __shfl_sync(0xffffffffu, h.splits[0], from);
        const int second = __shfl_sync(0xffffffffu, h.splits[1], from);
        w.b = 2 * from;
        if (left >= heads * splits) {
            left -= heads * splits;
            splits = second;
            ++w.b;
        }
        unit = w.on ? left / splits : 0;
        w.split = w.on ? left - unit * splits : 0;
        w.chunk = h.chunk;
    } else {
        unit = (int)blockIdx.x / a.splits;
        w.split = (int)blockIdx.x - unit * a.splits;
        const int heads = a.K * a.row_tiles;
        w.b = unit / heads;
        unit -= w.b * heads;
        w.chunk = 1 << 30;
        if (a.splits > 1) {
            const int vis = seen_by(a, w.b).vis;
            w.chunk = (((vis < 0 ? 0 : vis) + a.splits - 1) / a.splits + 63) / 64 * 64;
        }
    }
    w.kh = unit / a.row_tiles;
    w.rt = unit - w.kh * a.row_tiles;
    w.c0 = w.split * w.chunk;
    return w;
}

// A position's entry of the page table, read one tile before it is used: the
// read takes as long as a row's own.  off < 0: no position.
struct Entry {
    int id, off;
};
__device__ __forceinline__ Entry entry_of(const PagedArgs& a, const Seen& v, const int32_t* row, int t, bool on) {
    if (!on) return Entry{0, -1};
    const int tok = v.token(t), p = tok / a.page;
    return Entry{row[p], tok - p * a.page};
}
// Its place (page * page size + slot); -1 where there is no position or, with
// bad set, where the table names no page.
__device__ __forceinline__ int place_of(const PagedArgs& a, const Entry& e, bool& bad) {
    if (e.off < 0) return -1;
    if (e.id < 0 || e.id >= a.n_pages) {
        bad = true;
        return -1;
    }
    return e.id * a.page + e.off;
}

// The float at `p` of this block's shared memory in block `rank` of the cluster.
__device__ __forceinline__ float cluster_float(const float* p, int rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

constexpr int PG_CLUSTER = 8;  // splits that are joined in a cluster, at most

// Joins the warps' (m, l, sums) of one unit in shared memory, in warp order;
// then writes the output (one split), or this split's partial, or joins the
// splits of a cluster, in split order, each block a part of the outputs.
// ms, ls [PG_WARPS][R] (the joined ones in the first R); os [PG_WARPS][R][pitch].
template <typename T>
__device__ __forceinline__ void join_warps(const PagedArgs& a, float* ms, float* ls, float* os, int pitch, int rows,
                                           int b, int h0, int split, bool bad, bool none) {
    float* part = a.share ? a.part + blockIdx.x * part_floats(a.R, a.D) : nullptr;
    T* out = static_cast<T*>(a.o) + ((int64_t)b * a.H + h0) * a.D;
    for (int i = threadIdx.x; i < rows * a.D; i += PG_WARPS * 32) {
        const int r = i / a.D, d = i - r * a.D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < PG_WARPS; ++w) M = fmaxf(M, ms[w * a.R + r]);
        const float base = M == -INFINITY ? 0.f : M;
        float l = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < PG_WARPS; ++w) {
            const float f = exp2_fast(ms[w * a.R + r] - base);
            l = fmaf(ls[w * a.R + r], f, l);
            x = fmaf(os[(w * a.R + r) * pitch + d], f, x);
        }
        if (bad) l = __int_as_float(0x7fffffff);
        if (a.splits > 1) {
            os[r * pitch + d] = x;  // read by this thread alone
        } else if (part) {
            if (d == 0) {
                part[r] = M;
                part[a.R + r] = l;
            }
            part[2 * a.R + r * pad4(a.D) + d] = x;
        } else {
            out[i] = zg_from_float<T>(none ? 0.f : x / l);
        }
    }
    if (a.splits == 1) return;
    // the row's maximum and sum over the warps, by one warp's lanes (R <= 16)
    __syncthreads();
    if (threadIdx.x < a.R) {
        const int r = threadIdx.x;
        float M = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < PG_WARPS; ++w) M = fmaxf(M, ms[w * a.R + r]);
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < PG_WARPS; ++w) l = fmaf(ls[w * a.R + r], exp2_fast(ms[w * a.R + r] - base), l);
        ms[r] = M;  // read by this thread alone
        ls[r] = bad ? __int_as_float(0x7fffffff) : l;
    }
    cluster_sync_all();
    for (int i = split * PG_WARPS * 32 + threadIdx.x; i < rows * a.D; i += a.splits * PG_WARPS * 32) {
        const int r = i / a.D, d = i - r * a.D;
        float m[PG_CLUSTER], l[PG_CLUSTER], x[PG_CLUSTER], M = -INFINITY;
#pragma unroll
        for (int s = 0; s < PG_CLUSTER; ++s)
            if (s < a.splits) {
                m[s] = cluster_float(ms + r, s);
                l[s] = cluster_float(ls + r, s);
                x[s] = cluster_float(os + r * pitch + d, s);
                M = fmaxf(M, m[s]);
            }
        const float base = M == -INFINITY ? 0.f : M;
        float num = 0.f, den = 0.f;
#pragma unroll
        for (int s = 0; s < PG_CLUSTER; ++s)
            if (s < a.splits) {
                const float f = exp2_fast(m[s] - base);
                num = fmaf(x[s], f, num);
                den = fmaf(l[s], f, den);
            }
        out[i] = zg_from_float<T>(none ? 0.f : num / den);
    }
    cluster_sync_all();  // no block leaves while another reads its memory
}

// bf16 with D a multiple of 8 (padded to DP with zeros): up to 16 query heads
// of one key head are the rows of m16n8k16 products.  Every warp works alone
// on tiles of 16 positions, its own ring of STAGES tiles filled by cp.async
// (a tile's rows are fetched through the page table, whose entries are read
// one tile earlier), with its own running maximum and sum; the four warps
// meet once, at the end.  The products are a small part of the time the
// bytes take: 16 rows of which G are used cost nothing that matters, and a
// larger tile of the tensor cores of this chip would have to wait for 128
// positions where a warp goes on after 16.
template <int DP, int STAGES, bool SHARE>
__global__ void __launch_bounds__(PG_WARPS * 32) paged_mma_kernel(const PagedArgs a) {
    using T = __nv_bfloat16;
    constexpr int CPR = DP / 8;             // 16-byte chunks of a row
    constexpr int TILE = 16 * DP * 2;       // bytes of 16 key (or value) rows
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float ms[PG_WARPS * 16], ls[PG_WARPS * 16];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Work w = work_of<SHARE>(a);
    if (!w.on) return;
    const int b = w.b, kh = w.kh, rt = w.rt, c0 = w.c0;
    const int rows = a.G - rt * 16 < 16 ? a.G - rt * 16 : 16;
    const int h0 = kh * a.G + rt * 16;
    const Seen see = seen_by(a, b);
    const int end = see.vis - c0 < w.chunk ? see.vis : c0 + w.chunk;  // this block: [c0, end)
    const int32_t* table = a.table + (int64_t)b * a.max_pages;
    const int tiles_all = end > c0 ? (end - c0 + 15) / 16 : 0;
    const int tiles = tiles_all > warp ? (tiles_all - warp + PG_WARPS - 1) / PG_WARPS : 0;
    uint8_t* ring = smem + warp * (STAGES * 2 * TILE);
    const T* kp = static_cast<const T*>(a.kp) + kh * a.D;
    const T* vp = static_cast<const T*>(a.vp) + kh * a.D;
    const int64_t token_pitch = (int64_t)a.K * a.D;
    bool bad = false;

    // lanes 0..15: the table's entry for each row of this warp's tile i
    auto entries = [&](int i) {
        const int t = c0 + (warp + PG_WARPS * i) * 16 + lane;
        return entry_of(a, see, table, t, i < tiles && lane < 16 && t < end);
    };
    auto fetch = [&](int stage, int place) {
        const uint32_t kd = shared_u32(ring + stage * 2 * TILE), vd = kd + TILE;
#pragma unroll
        for (int it = 0; it < CPR / 2; ++it) {
            const int i = it * 32 + lane, r = i / CPR, c = i % CPR;
            const int at = __shfl_sync(0xffffffffu, place, r);
            const bool on = at >= 0 && c * 8 < a.D;
            const int64_t off = on ? at * token_pitch + c * 8 : 0;
            const uint32_t to = r * (DP * 2) + ((c ^ (r & 7)) * 16);
            copy16(kd + to, kp + off, on ? 16 : 0);
            copy16(vd + to, vp + off, on ? 16 : 0);
        }
    };

    Entry entry = entries(0);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        const Entry next = entries(s + 1);
        if (s < tiles) fetch(s, place_of(a, entry, bad));
        copy_commit();
        entry = next;
    }

    // queries as the rows of A: (row, k) = (lane / 4 [+ 8], 2 (lane % 4) [+ 8]) in k-steps of 16
    uint32_t qf[DP / 16][4];
    {
        const T* q = static_cast<const T*>(a.q) + b * a.ldq + (int64_t)h0 * a.D;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = lane / 4 + (e & 1) * 8, d = k * 16 + (lane % 4) * 2 + (e >> 1) * 8;
                qf[k][e] = r < rows && d < a.D ? *reinterpret_cast<const uint32_t*>(q + (int64_t)r * a.D + d) : 0u;
            }
    }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // rows lane/4 and lane/4 + 8, in units of log2

    const int k_row = (lane % 8) + 8 * (lane / 16), k_chunk = (lane / 8) % 2;
    const int v_row = (lane % 8) + 8 * ((lane / 8) % 2), v_chunk = lane / 16;
    for (int i = 0; i < tiles; ++i) {
        copy_wait<STAGES - 2>();
        __syncwarp();  // every lane's copies of tile i have landed, and tile i-1 has been read
        {
            const Entry next = entries(i + STAGES);
            if (i + STAGES - 1 < tiles) fetch((i + STAGES - 1) % STAGES, place_of(a, entry, bad));
            copy_commit();
            entry = next;
        }
        const uint32_t kt = shared_u32(ring + (i % STAGES) * 2 * TILE), vt = kt + TILE;
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            uint32_t f[4];
            ldmatrix4(f, kt + k_row * (DP * 2) + (((2 * k + k_chunk) ^ (k_row & 7)) * 16));
            mma_bf16(s[0], qf[k], f[0], f[1]);
            mma_bf16(s[1], qf[k], f[2], f[3]);
        }
        const int t0 = c0 + (warp + PG_WARPS * i) * 16;
        float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[j][e] = t0 + j * 8 + (lane % 4) * 2 + (e & 1) < end ? s[j][e] * a.scale : -INFINITY;
                if (e < 2) n0 = fmaxf(n0, s[j][e]);
                else n1 = fmaxf(n1, s[j][e]);
            }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
        }
        n0 = fmaxf(n0, m0);
        n1 = fmaxf(n1, m1);
        const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
        if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
            const float f0 = exp2_fast(m0 - b0), f1 = exp2_fast(m1 - b1);
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int d = 0; d < DP / 8; ++d) {
                o[d][0] *= f0;
                o[d][1] *= f0;
                o[d][2] *= f1;
                o[d][3] *= f1;
            }
            m0 = n0;
            m1 = n1;
        }
        // weights, rounded to bf16 as the second product's operand (their sum
        // is of the unrounded ones): half a step of each weight, 2^-9
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float p0 = exp2_fast(s[j][0] - b0), p1 = exp2_fast(s[j][1] - b0);
            const float p2 = exp2_fast(s[j][2] - b1), p3 = exp2_fast(s[j][3] - b1);
            l0 += p0 + p1;
            l1 += p2 + p3;
            p[2 * j] = pack_bf16(p0, p1);
            p[2 * j + 1] = pack_bf16(p2, p3);
        }
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            uint32_t f[4];
            ldmatrix4_t(f, vt + v_row * (DP * 2) + (((2 * d + v_chunk) ^ (v_row & 7)) * 16));
            mma_bf16(o[2 * d], p, f[0], f[1]);
            mma_bf16(o[2 * d + 1], p, f[2], f[3]);
        }
    }
    copy_wait<0>();
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, x);
        l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    bad = __syncthreads_or(bad || see.vis < 0);  // the rings are free from here on
    float* os = reinterpret_cast<float*>(smem);  // [PG_WARPS][16][DP]
    const int r = lane / 4;
    if (lane % 4 == 0) {
        ms[warp * 16 + r] = m0;
        ms[warp * 16 + r + 8] = m1;
        ls[warp * 16 + r] = l0;
        ls[warp * 16 + r + 8] = l1;
    }
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) {
        float* to = os + (warp * 16 + r) * DP + d * 8 + (lane % 4) * 2;
        *reinterpret_cast<float2*>(to) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(to + 8 * DP) = make_float2(o[d][2], o[d][3]);
    }
    __syncthreads();
    join_warps<T>(a, ms, ls, os, DP, rows, b, h0, w.split, bad, see.vis == 0);
}

// Any type, width and alignment, in float32 on the FMA pipe.  A warp's tile
// has 32 / PARTS positions: PARTS lanes share a position's dot products (each
// a PARTS-th of the columns), then every lane takes the columns lane + 32 i
// of the sums.  GT query heads at a time; the same ring of tiles as above,
// its rows kept as they are stored, 16 bytes apart from the next one's banks.
constexpr int PG_FMA_STAGES = 2;  // three blocks an SM (two with 3: a batch of 64 x 1000 in float32 34.2 us, not 32.6)

template <typename T, int PARTS, int GT, bool SHARE>
__global__ void __launch_bounds__(PG_WARPS * 32) paged_fma_kernel(const PagedArgs a, int vec) {
    constexpr int TT = 32 / PARTS, STAGES = PG_FMA_STAGES, NI = PARTS, DMAX = 32 * PARTS;
    constexpr int PITCH = DMAX * (int)sizeof(T) + 16, TILE = TT * PITCH;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float ms[PG_WARPS * GT], ls[PG_WARPS * GT];
    __shared__ __align__(16) float qs[GT][36 * PARTS];  // parts of 32 columns, 4 banks apart
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Work w = work_of<SHARE>(a);
    if (!w.on) return;
    const int b = w.b, kh = w.kh, rt = w.rt, c0 = w.c0;
    const int rows = a.G - rt * GT < GT ? a.G - rt * GT : GT;
    const int h0 = kh * a.G + rt * GT;
    const Seen see = seen_by(a, b);
    const int end = see.vis - c0 < w.chunk ? see.vis : c0 + w.chunk;
    const int32_t* table = a.table + (int64_t)b * a.max_pages;
    const int tiles_all = end > c0 ? (end - c0 + TT - 1) / TT : 0;
    const int tiles = tiles_all > warp ? (tiles_all - warp + PG_WARPS - 1) / PG_WARPS : 0;
    uint8_t* ring = smem + warp * (STAGES * 2 * TILE);
    const T* kp = static_cast<const T*>(a.kp) + kh * a.D;
    const T* vp = static_cast<const T*>(a.vp) + kh * a.D;
    const int64_t token_pitch = (int64_t)a.K * a.D;
    bool bad = false;

    for (int i = threadIdx.x; i < GT * DMAX; i += PG_WARPS * 32) {
        const int r = i / DMAX, d = i % DMAX;
        qs[r][d / 32 * 36 + d % 32] = r < rows && d < a.D ? zg_to_float(static_cast<const T*>(a.q)[b * a.ldq + (int64_t)(h0 + r) * a.D + d]) * a.scale : 0.f;
    }
    // the columns past D stay zero in every stage
    for (int i = lane; i < STAGES * 2 * TILE / 4; i += 32) reinterpret_cast<uint32_t*>(ring)[i] = 0u;
    __syncthreads();

    auto entries = [&](int i) {
        const int t = c0 + (warp + PG_WARPS * i) * TT + lane;
        return entry_of(a, see, table, t, i < tiles && lane < TT && t < end);
    };
    auto fetch = [&](int stage, int place) {
        uint8_t* kd = ring + stage * 2 * TILE;
        uint8_t* vd = kd + TILE;
        if (vec) {
            // 16-byte words of the padded rows, zeros behind D
            constexpr int N = 16 / sizeof(T), WORDS = DMAX / N;
#pragma unroll
            for (int it = 0; it < TT * WORDS / 32; ++it) {
                const int i = it * 32 + lane, r = i / WORDS, c = i % WORDS;
                const int at = __shfl_sync(0xffffffffu, place, r);
                const bool on = at >= 0 && c * N < a.D;
                const int64_t off = on ? at * token_pitch + c * N : 0;
                copy16(shared_u32(kd + r * PITCH + c * 16), kp + off, on ? 16 : 0);
                copy16(shared_u32(vd + r * PITCH + c * 16), vp + off, on ? 16 : 0);
            }
        } else {
            for (int r = 0; r < TT; ++r) {
                const int at = __shfl_sync(0xffffffffu, place, r);
                const int64_t off = at >= 0 ? at * token_pitch : 0;
                for (int c = lane; c < a.D; c += 32) {
                    reinterpret_cast<T*>(kd + r * PITCH)[c] = at >= 0 ? kp[off + c] : zg_from_float<T>(0.f);
                    reinterpret_cast<T*>(vd + r * PITCH)[c] = at >= 0 ? vp[off + c] : zg_from_float<T>(0.f);
                }
            }
        }
    };
    Entry entry = entries(0);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        const Entry next = entries(s + 1);
        if (s < tiles) fetch(s, place_of(a, entry, bad));
        copy_commit();
        entry = next;
    }
    float o[GT][NI], m[GT], l[GT];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) o[g][i] = 0.f;
    }
    const int tok = lane % TT, part = lane / TT;
    for (int i = 0; i < tiles; ++i) {
        copy_wait<STAGES - 2>();
        __syncwarp();
        {
            const Entry next = entries(i + STAGES);
            if (i + STAGES - 1 < tiles) fetch((i + STAGES - 1) % STAGES, place_of(a, entry, bad));
            copy_commit();
            entry = next;
        }
        const uint8_t* kt = ring + (i % STAGES) * 2 * TILE;
        const uint8_t* vt = kt + TILE;
        float s[GT];
#pragma unroll
        for (int g = 0; g < GT; ++g) s[g] = 0.f;
        const T* kr = reinterpret_cast<const T*>(kt + tok * PITCH) + part * 32;
#pragma unroll
        for (int d = 0; d < 32; d += 4) {
            float kv[4];
            if constexpr (sizeof(T) == 4) {
                const float4 x = *reinterpret_cast<const float4*>(kr + d);
                kv[0] = x.x; kv[1] = x.y; kv[2] = x.z; kv[3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(kr + d);
                kv[0] = __uint_as_float(x.x << 16); kv[1] = __uint_as_float(x.x & 0xffff0000u);
                kv[2] = __uint_as_float(x.y << 16); kv[3] = __uint_as_float(x.y & 0xffff0000u);
            }
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const float4 x = *reinterpret_cast<const float4*>(&qs[g][part * 36 + d]);
                s[g] = fmaf(kv[0], x.x, fmaf(kv[1], x.y, fmaf(kv[2], x.z, fmaf(kv[3], x.w, s[g]))));
            }
        }
        const bool on = c0 + (warp + PG_WARPS * i) * TT + tok < end;
#pragma unroll
        for (int g = 0; g < GT; ++g) {
#pragma unroll
            for (int x = TT; x < 32; x <<= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], x);
            s[g] = on ? s[g] : -INFINITY;
            float n = s[g];
#pragma unroll
            for (int x = 1; x < TT; x <<= 1) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, x));
            n = fmaxf(n, m[g]);
            const float base = n == -INFINITY ? 0.f : n;
            const float f = exp2f(m[g] - base);
            m[g] = n;
            s[g] = exp2f(s[g] - base);
            l[g] = fmaf(l[g], f, part == 0 ? s[g] : 0.f);
#pragma unroll
            for (int c = 0; c < NI; ++c) o[g][c] *= f;
        }
#pragma unroll 4
        for (int t = 0; t < TT; ++t) {
            float v[NI];
            const T* vr = reinterpret_cast<const T*>(vt + t * PITCH);
#pragma unroll
            for (int c = 0; c < NI; ++c) v[c] = zg_to_float(vr[lane + 32 * c]);
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const float p = __shfl_sync(0xffffffffu, s[g], t);
#pragma unroll
                for (int c = 0; c < NI; ++c) o[g][c] = fmaf(p, v[c], o[g][c]);
            }
        }
    }
    copy_wait<0>();
    bad = __syncthreads_or(bad || see.vis < 0);
    float* os = reinterpret_cast<float*>(smem);  // [PG_WARPS][GT][DMAX]
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], x);
        if (lane == 0) {
            ms[warp * GT + g] = m[g];
            ls[warp * GT + g] = l[g];
        }
#pragma unroll
        for (int c = 0; c < NI; ++c) os[(warp * GT + g) * DMAX + lane + 32 * c] = o[g][c];
    }
    __syncthreads();
    join_warps<T>(a, ms, ls, os, DMAX, rows, b, h0, w.split, bad, see.vis == 0);
}

// Joins the splits of one query head: a block per (b, h), its warps over the
// splits, summed in warp order.  It is launched so that its blocks start as
// the splits' last one ends.  (With its blocks waiting in their places while
// the splits run, one sequence of 131000 takes 54.3 us instead of 51.6.)
template <typename T>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedArgs a) {
    __shared__ float4 sums[8][64];
    __shared__ float sum_l[8];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int b = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x % a.H);
    const int kh = h / a.G, rt = h % a.G / a.R, r = h % a.G % a.R;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched before the splits' kernel has ended
    const int vis = seen_by(a, b).vis;
    const Shares shares = shares_of(a);
    const int even = __shfl_sync(0xffffffffu, shares.splits[0], b / 2), odd = __shfl_sync(0xffffffffu, shares.splits[1], b / 2);
    const int n = b % 2 ? odd : even;  // shares of this unit, from block `first`
    const int first = __shfl_sync(0xffffffffu, shares.before, b / 2) + (b % 2 ? a.K * a.row_tiles * even : 0) +
                      (kh * a.row_tiles + rt) * n;
    const int64_t pf = part_floats(a.R, a.D);
    const float* part = a.part + first * pf;
    const int words = pad4(a.D) / 4;
    float M = -INFINITY;
    for (int s = lane; s < n; s += 32) M = fmaxf(M, part[s * pf + r]);
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float base = M == -INFINITY ? 0.f : M;
    float l = 0.f;
    float4 x[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
    for (int s = warp; s < n; s += 8) {
        const float* p = part + s * pf;
        const float f = exp2f(p[r] - base);
        l = fmaf(p[a.R + r], f, l);
        const float* row = p + 2 * a.R + r * (words * 4);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (lane + 32 * j < words) {
                // rows start on 8-byte boundaries at least (2 R floats, R even, or R = 1)
                const float2 u = *reinterpret_cast<const float2*>(row + 4 * (lane + 32 * j));
                const float2 w = *reinterpret_cast<const float2*>(row + 4 * (lane + 32 * j) + 2);
                x[j].x = fmaf(u.x, f, x[j].x);
                x[j].y = fmaf(u.y, f, x[j].y);
                x[j].z = fmaf(w.x, f, x[j].z);
                x[j].w = fmaf(w.y, f, x[j].w);
            }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (lane + 32 * j < words) sums[warp][lane + 32 * j] = x[j];
    if (lane == 0) sum_l[warp] = l;
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= a.D) return;
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        num += reinterpret_cast<const float*>(sums[w])[d];
        den += sum_l[w];
    }
    const float out = vis < 0 ? __int_as_float(0x7fffffff) : vis == 0 ? 0.f : num / den;
    static_cast<T*>(a.o)[((int64_t)b * a.H + h) * a.D + d] = zg_from_float<T>(out);
}

// How a call is cut: R query rows of a unit, the units' splits, or the blocks
// that share them.
struct PagedPlan {
    int R, row_tiles, splits, share;
    bool mma;
};

PagedPlan paged_plan(int64_t B, int H, int K, int D, int64_t longest, int window, int sinks, int dtype) {
    PagedPlan p{};
    const int G = H / K;
    p.mma = dtype == ZG_BF16 && D % 8 == 0;
    p.R = p.mma ? 16 : G == 1 ? 1 : G <= 4 ? 4 : 8;
    p.row_tiles = (G + p.R - 1) / p.R;
    int64_t vis = longest;
    if (window > 0 && (int64_t)window + sinks < vis) vis = (int64_t)window + sinks;
    const int64_t units = B * K * p.row_tiles, blocks = (p.mma ? 2 : 3) * 148;
    // Two blocks run on each of 148 SMs (three of the FMA path): as many splits
    // as fill them once.  (Four times as many, so that a batch of 64 sequences
    // of different lengths evens out, was 126 us instead of 81: a block costs
    // its pipeline's filling and its part in the join.)  Up to PG_CLUSTER
    // splits are a cluster of two, four or eight blocks, which joins them by
    // itself and whose blocks have equal parts of what its unit sees.  Units
    // that would be cut further are shared out to all blocks by the lengths
    // that the device knows, and a kernel of its own joins them.  (Split by the
    // table's width instead, a sequence of 8000 in a table of 131072 took 42
    // us, now 12.2; 8 of 1000 in a table of 16384 26 us, now 11.2.)
    int64_t splits = (blocks + units - 1) / units;
    if (splits > (vis + PG_MIN_CHUNK - 1) / PG_MIN_CHUNK) splits = (vis + PG_MIN_CHUNK - 1) / PG_MIN_CHUNK;
    p.splits = 1;
    if (splits > PG_CLUSTER)
        p.share = (int)blocks;  // more than twice the units, of which there are less than 64
    else if (splits > 1)
        p.splits = splits <= 2 ? 2 : splits <= 4 ? 4 : 8;
    return p;
}

size_t paged_workspace(const PagedPlan& p, int D) { return (size_t)(p.share * part_floats(p.R, D)) * sizeof(float); }

bool paged_sizes_ok(int64_t n_pages, int page, int64_t B, int H, int K, int D, int max_pages) {
    return n_pages >= 0 && page >= 1 && B >= 0 && H >= 1 && K >= 1 && D >= 1 && max_pages >= 0 && H % K == 0 &&
           B <= INT32_MAX / H;
}

template <typename F>
int set_smem(F* f, size_t bytes) {
    if (cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
        return zg::fail(ZG_ERR_CUDA, "zg_paged_attention: shared memory attribute");
    return ZG_OK;
}

template <typename... P, typename... A>
int launch_split(void (*f)(P...), const PagedArgs& a, int64_t blocks, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)blocks);
    c.blockDim = dim3(PG_WARPS * 32);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)a.splits;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = a.splits > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&c, f, args...);
    if (e != cudaSuccess) return zg::fail(ZG_ERR_CUDA, "zg_paged_attention: %s", cudaGetErrorString(e));
    return zg::check_launch("zg_paged_attention");
}

template <int DP, int STAGES>
int launch_mma(const PagedArgs& a, int64_t blocks, cudaStream_t st) {
    const size_t smem = (size_t)PG_WARPS * STAGES * 2 * 16 * DP * 2;
    const auto f = a.share ? paged_mma_kernel<DP, STAGES, true> : paged_mma_kernel<DP, STAGES, false>;
    if (int rc = set_smem(f, smem)) return rc;
    zg::LaunchTimer zg_lt_("paged_attention", st);
    return launch_split(f, a, blocks, smem, st, a);
}

template <typename T, int PARTS, int GT>
int launch_fma(const PagedArgs& a, int vec, int64_t blocks, cudaStream_t st) {
    const size_t ring = (size_t)PG_WARPS * PG_FMA_STAGES * 2 * (32 / PARTS) * (32 * PARTS * sizeof(T) + 16);
    const size_t out = (size_t)PG_WARPS * GT * 32 * PARTS * sizeof(float);
    const size_t smem = ring > out ? ring : out;
    const auto f = a.share ? paged_fma_kernel<T, PARTS, GT, true> : paged_fma_kernel<T, PARTS, GT, false>;
    if (int rc = set_smem(f, smem)) return rc;
    zg::LaunchTimer zg_lt_("paged_attention_fma", st);
    return launch_split(f, a, blocks, smem, st, a, vec);
}

template <typename T, int PARTS>
int launch_fma_rows(const PagedArgs& a, int vec, int64_t blocks, cudaStream_t st) {
    if (a.R == 1) return launch_fma<T, PARTS, 1>(a, vec, blocks, st);
    if (a.R == 4) return launch_fma<T, PARTS, 4>(a, vec, blocks, st);
    return launch_fma<T, PARTS, 8>(a, vec, blocks, st);
}

template <typename T>
int launch_fma_any(const PagedArgs& a, int vec, int64_t blocks, cudaStream_t st) {
    if (a.D <= 64) return launch_fma_rows<T, 2>(a, vec, blocks, st);
    if (a.D <= 128) return launch_fma_rows<T, 4>(a, vec, blocks, st);
    return launch_fma_rows<T, 8>(a, vec, blocks, st);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int zg_append_pages(void* k_pages, void* v_pages, int64_t n_pages, int page, int K, int D, const void* k,
                               int64_t ldk, const void* v, int64_t ldv, int64_t B, int64_t S, const int32_t* table,
                               int max_pages, const int32_t* lengths, const int32_t* counts, int dtype,
                               int32_t* new_lengths, void* stream) {
    if (!paged_sizes_ok(n_pages, page, B, K, K, D, max_pages) || S < 0 || B > INT32_MAX || S > INT32_MAX)
        return zg::fail(ZG_ERR_INVALID, "zg_append_pages: bad sizes");
    if (ldk < (int64_t)K * D || ldv < (int64_t)K * D)
        return zg::fail(ZG_ERR_INVALID, "zg_append_pages: row pitch below K*D");
    if (!zg::dtype_ok(dtype)) return zg::fail(ZG_ERR_INVALID, "zg_append_pages: bad dtype");
    if ((int64_t)max_pages * page > PG_MOST) return zg::fail(ZG_ERR_INVALID, "zg_append_pages: table too long");
    if (B == 0) return ZG_OK;
    if (!lengths || !new_lengths || (max_pages && !table) || (S && (!k || !v)) || (n_pages && (!k_pages || !v_pages)))
        return zg::fail(ZG_ERR_INVALID, "zg_append_pages: null pointer");
    const int64_t blocks = (B * S + B + 7) / 8;
    if (blocks > INT32_MAX) return zg::fail(ZG_ERR_INVALID, "zg_append_pages: too many tokens");
    const int esize = (int)zg::dtype_size(dtype);
    const int n = 16 / esize;
    const int64_t row = (int64_t)K * D;
    const bool vec = row % n == 0 && ldk % n == 0 && ldv % n == 0 && aligned16(k) && aligned16(v) &&
                     aligned16(k_pages) && aligned16(v_pages);
    const int w = vec ? n : 1;
    const AppendArgs a{k_pages, v_pages, k, v, table, lengths, counts, new_lengths, n_pages, ldk / w, ldv / w,
                       row / w, B * S, page, max_pages, (int)B, (int)S};
    cudaStream_t st = zg::as_stream(stream);
    zg::LaunchTimer zg_lt_("append_pages", st);
    if (vec)
        append_kernel<uint4><<<(unsigned)blocks, 256, 0, st>>>(a);
    else if (esize == 2)
        append_kernel<uint16_t><<<(unsigned)blocks, 256, 0, st>>>(a);
    else
        append_kernel<uint32_t><<<(unsigned)blocks, 256, 0, st>>>(a);
    return zg::check_launch("zg_append_pages");
}

extern "C" size_t zg_paged_attention_workspace_size(int64_t B, int H, int K, int D, int max_pages, int page,
                                                    int window, int sinks, int dtype) {
    if (!paged_sizes_ok(0, page, B, H, K, D, max_pages) || B == 0 || D > 256 || window < 0 || sinks < 0 ||
        !zg::dtype_ok(dtype))
        return 0;
    return paged_workspace(paged_plan(B, H, K, D, (int64_t)max_pages * page, window, sinks, dtype), D);
}

extern "C" int zg_paged_attention(const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                                  int64_t n_pages, int page, const int32_t* table, int max_pages,
                                  const int32_t* lengths, int64_t B, int H, int K, int D, int window, int sinks,
                                  int dtype, void* o, void* workspace, size_t workspace_bytes, void* stream) {
    if (!paged_sizes_ok(n_pages, page, B, H, K, D, max_pages))
        return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: bad sizes");
    if (D > 256) return zg::fail(ZG_ERR_UNSUPPORTED, "zg_paged_attention: head dim above 256");
    if (window < 0 || sinks < 0) return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: window and sinks must be >= 0");
    if (ldq < (int64_t)H * D) return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: row pitch below H*D");
    if (!zg::dtype_ok(dtype)) return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: bad dtype");
    if ((int64_t)max_pages * page > PG_MOST || (n_pages && n_pages > PG_MOST / page))
        return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: more positions than 32 bits count");
    if (B == 0) return ZG_OK;
    if (!q || !lengths || !o || (max_pages && !table) || (n_pages && (!k_pages || !v_pages)))
        return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: null pointer");
    PagedPlan p = paged_plan(B, H, K, D, (int64_t)max_pages * page, window, sinks, dtype);
    const size_t need = paged_workspace(p, D);
    if (need && (!workspace || workspace_bytes < need))
        return zg::fail(ZG_ERR_WORKSPACE, "zg_paged_attention: workspace of %zu bytes needed", need);
    const int64_t blocks = p.share ? p.share : B * K * p.row_tiles * p.splits;
    if (blocks > INT32_MAX) return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: too many rows");
    const int n = 16 / (int)zg::dtype_size(dtype);
    const int vec = D % n == 0 && aligned16(k_pages) && aligned16(v_pages);
    PagedArgs a{q, k_pages, v_pages, table, lengths, o, static_cast<float*>(workspace), ldq, n_pages, page, max_pages,
                (int)B, H, K, D, H / K, p.row_tiles, p.R, window, sinks, p.splits, p.share,
                (float)(1.4426950408889634 / sqrt((double)D))};
    cudaStream_t st = zg::as_stream(stream);
    int rc;
    if (p.mma && vec && ldq % 2 == 0 && (reinterpret_cast<uintptr_t>(q) & 3) == 0) {
        rc = D <= 64 ? launch_mma<64, 4>(a, blocks, st)
             : D <= 128 ? launch_mma<128, 3>(a, blocks, st) : launch_mma<256, 3>(a, blocks, st);
    } else if (p.mma) {
        return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: bf16 pages with D a multiple of 8 must be 16-byte "
                                        "aligned, q 4-byte aligned with an even pitch");
    } else {
        rc = dtype == ZG_BF16 ? launch_fma_any<__nv_bfloat16>(a, vec, blocks, st)
                              : launch_fma_any<float>(a, vec, blocks, st);
    }
    if (rc != ZG_OK || !p.share) return rc;
    zg::LaunchTimer zg_lt_("paged_join", st);
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(B * H));
    c.blockDim = dim3(256);
    c.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&c, dtype == ZG_BF16 ? paged_join_kernel<__nv_bfloat16> : paged_join_kernel<float>, a);
    if (e != cudaSuccess) return zg::fail(ZG_ERR_CUDA, "zg_paged_attention: %s", cudaGetErrorString(e));
    return zg::check_launch("zg_paged_attention");
}
