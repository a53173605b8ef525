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
// How a sequence is cut is a matter of what it sees and of the heads alone, so
// that its result has the same bits whatever else is in the launch (another
// candidate's sequences, a wider table): into n chunks of its visible
// positions, whose tiles the four warps take by turns.  A warp has a maximum,
// a sum and outputs of its own for each chunk; those of one warp are folded
// chunk after chunk, and the four warps' joined behind that.  How many chunks
// a block takes is a matter of the launch:
//   whole:   a block takes a unit (a sequence, a key head and up to 16 of its
//            query heads), its warps fold chunk after chunk as they go;
//   cluster: a unit's chunks are one block each of a cluster, which folds them;
//   share:   blocks take runs of chunks, a kernel of its own folds them: equal
//            parts of a unit's, or where there are few units runs of about as
//            many positions, by the lengths that the device knows.
// (The four warps joined at each chunk's end, which is less to keep, makes them
// wait for one another: 64 sequences of 1000 to 4000 took 95 us.)
struct PagedArgs {
    const void *q, *kp, *vp;
    const int32_t *table, *lengths;
    void* o;
    float* part;  // of each unit, chunk and warp, P rows of sums, then m [P], l [P]; null where blocks join by themselves
    int64_t ldq, n_pages;
    // R: query rows of a unit (heads that share a key head), P: those that there are
    int page, max_pages, B, H, K, D, G, row_tiles, R, P;
    // splits: the blocks of a unit (a cluster unless part is set); share > 0: so many blocks of all units instead
    int window, sinks, splits, share;
    int each, most;  // chunks of a sequence: at most, and at most in this launch
    int least;       // positions of a chunk where there are more than 8 PG_CHUNK, at least
    float scale;     // log2(e) / sqrt(D)
};

__host__ __device__ __forceinline__ int pad4(int d) { return (d + 3) / 4 * 4; }
__host__ __device__ __forceinline__ int64_t part_floats(int P, int D) { return ((int64_t)P * (pad4(D) + 2) + 3) / 4 * 4; }

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

constexpr int PG_CHUNK = 128;  // positions of a chunk at least: less would be the pipeline's filling and the join

// Positions of a chunk of `vis`, a multiple of 64.  Above the eight chunks of
// a cluster those of the tensor-core kernel are twice as long at least, as
// each costs a whole unit's warps their fold: 64 sequences of 1000 to 4000 take
// 83 us with 256, 86 with 128 (and 81 cut not at all); one of 8000 over 12
// heads 11.5, with 512 14.9.  (float32's products take longer for the same
// bytes: 2 sequences of 9000, 10 heads of one key head, 22 us with 128, 28 with 256.)
__device__ __forceinline__ int chunk_of(const PagedArgs& a, int vis) {
    const int even = (vis + a.each - 1) / a.each, least = vis <= 8 * PG_CHUNK ? PG_CHUNK : a.least;
    return ((even < least ? least : even) + 63) / 64 * 64;
}
__device__ __forceinline__ int chunks_of(const PagedArgs& a, int vis) {
    if (vis <= 0) return 0;
    const int chunk = chunk_of(a, vis);
    return (vis + chunk - 1) / chunk;
}

// The blocks of each unit, from the lengths of at most 64 sequences, so that
// each has about as many positions: lane l has those of sequences 2 l and
// 2 l + 1.
struct Shares {
    int n[2], blocks[2], before;  // chunks and blocks of a unit; blocks of the sequences before 2 l
};
__device__ __forceinline__ Shares shares_of(const PagedArgs& a) {
    const int lane = threadIdx.x % 32, heads = a.K * a.row_tiles;
    Shares h;
    int vis[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int v = 2 * lane + j < a.B ? seen_by(a, 2 * lane + j).vis : 0;
        vis[j] = v > 0 ? v : 0;
        h.n[j] = chunks_of(a, v);
    }
    long long total = (long long)vis[0] + vis[1];
#pragma unroll
    for (int f = 1; f < 32; f <<= 1) total += __shfl_xor_sync(0xffffffffu, total, f);
    total *= heads;
    auto used = [&](int positions) {  // blocks, if each takes so many
        int x = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int blocks = (int)((vis[j] + (unsigned)positions - 1) / (unsigned)positions);
            h.blocks[j] = blocks < h.n[j] ? blocks : h.n[j];
            x += h.blocks[j];
        }
#pragma unroll
        for (int f = 1; f < 32; f <<= 1) x += __shfl_xor_sync(0xffffffffu, x, f);
        return heads * x;
    };
    // the fewest positions that there are blocks for: from those if all were
    // full, a quarter of the way at a time, to those if each unit's last is not
    const int lo = (int)(total / a.share) + 1, hi = (int)(total / (a.share - a.B * heads)) + 1;
#pragma unroll 1
    for (int k = 0; k <= 4; ++k)
        if (used(lo + (int)((long long)(hi - lo) * k / 4)) <= a.share) break;
    const int mine = heads * (h.blocks[0] + h.blocks[1]);
    h.before = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, h.before, x);
        if (lane >= x) h.before += below;
    }
    h.before -= mine;
    return h;
}

// Weights are taken 2^-lift times smaller, so that no sum of `vis` finite
// values overflows on its way (the quotient is the same).
__device__ __forceinline__ int lift_of(int vis) { return 33 - __clz(vis > 0 ? vis : 1); }

// What this block does: chunks c0 .. c1 - 1 of row tile rt of key head kh of
// sequence b, its visible positions first .. end - 1; n: the sequence's chunks.
// on: it has any part.
struct Work {
    int b, kh, rt, c0, c1, n, chunk, first, end;
    bool on;
    // (of a whole unit known without the chunks, whose two quotients are formed
    // while the first rows are on their way)
    __device__ __forceinline__ void positions(const PagedArgs& a, int vis, bool whole) {
        first = 0;
        end = vis;
        if (whole) return;
        chunks(a, vis, false);
        first = c0 * chunk;
        if (c1 < n) end = c1 * chunk;
    }
    __device__ __forceinline__ void chunks(const PagedArgs& a, int vis, bool whole) {
        chunk = chunk_of(a, vis > 0 ? vis : 0);
        n = vis > 0 ? (vis + chunk - 1) / chunk : 0;
        if (whole) c1 = n;
        if (c1 > n) c1 = n;
    }
};
// (SHARE, with leaves in the workspace, is an instance of its own: with both
// in one, 64 sequences took 80.1 us instead of 77.9 before there were leaves.)
template <bool SHARE>
__device__ __forceinline__ Work work_of(const PagedArgs& a) {
    Work w;
    const int heads = a.K * a.row_tiles;
    int unit;  // of its sequence
    w.on = true;
    if (SHARE && a.share > 0) {
        const int x = (int)blockIdx.x;
        const Shares h = shares_of(a);
        const int mine = heads * (h.blocks[0] + h.blocks[1]);
        const unsigned found = __ballot_sync(0xffffffffu, x >= h.before && x < h.before + mine);
        w.on = found != 0;
        if (!w.on) return w;
        const int from = __ffs(found) - 1;
        int left = x - __shfl_sync(0xffffffffu, h.before, from);
        int blocks = __shfl_sync(0xffffffffu, h.blocks[0], from), n = __shfl_sync(0xffffffffu, h.n[0], from);
        const int blocks1 = __shfl_sync(0xffffffffu, h.blocks[1], from), n1 = __shfl_sync(0xffffffffu, h.n[1], from);
        w.b = 2 * from;
        if (left >= heads * blocks) {
            left -= heads * blocks;
            blocks = blocks1;
            n = n1;
            ++w.b;
        }
        unit = left / blocks;
        left -= unit * blocks;
        w.c0 = n * left / blocks;
        w.c1 = n * (left + 1) / blocks;
    } else {
        unit = (int)blockIdx.x / a.splits;
        const int at = (int)blockIdx.x - unit * a.splits;
        w.b = unit / heads;
        unit -= w.b * heads;
        w.c0 = at;  // the blocks of a cluster have a chunk each
        w.c1 = at + 1;
        if (SHARE) {
            const int n = chunks_of(a, seen_by(a, w.b).vis);
            w.c0 = n * at / a.splits;
            w.c1 = n * (at + 1) / a.splits;
        }
    }
    w.kh = unit / a.row_tiles;
    w.rt = unit - w.kh * a.row_tiles;
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
    __syncwarp();  // the barrier below is a converged warp's
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

constexpr int PG_CLUSTER = 8;  // chunks that a cluster folds, at most

// One more chunk (m, l, and of a column x) onto those before (M, L, X).  The
// same operations wherever it is done.
struct Fold {
    float before, next;  // factors of those before, and of the chunk
    __device__ __forceinline__ Fold(float& M, float& L, float m, float l) {
        const float n = fmaxf(M, m), base = n == -INFINITY ? 0.f : n;
        before = exp2f(M - base);
        next = exp2f(m - base);
        L = __fmaf_rn(l, next, __fmul_rn(L, before));
        M = n;
    }
    __device__ __forceinline__ float operator()(float X, float x) const { return __fmaf_rn(x, next, __fmul_rn(X, before)); }
};
// The four warps' (M, L) of a row: their factors and the sum.
struct Warps {
    float f[PG_WARPS], L;
    __device__ __forceinline__ Warps(const float (&M)[PG_WARPS], const float (&l)[PG_WARPS]) {
        const float m = fmaxf(fmaxf(M[0], M[1]), fmaxf(M[2], M[3])), base = m == -INFINITY ? 0.f : m;
        L = 0.f;
#pragma unroll
        for (int w = 0; w < PG_WARPS; ++w) {
            f[w] = exp2f(M[w] - base);
            L = __fmaf_rn(l[w], f[w], L);
        }
    }
    __device__ __forceinline__ float operator()(const float (&X)[PG_WARPS]) const {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < PG_WARPS; ++w) x = __fmaf_rn(X[w], f[w], x);
        return x / L;
    }
};

// The leaf of this warp in chunk c (its maximum, sum and outputs): where it goes in the workspace.
__device__ __forceinline__ float* leaf_of(const PagedArgs& a, const Work& w, int c) {
    return a.part + ((((int64_t)w.b * a.K + w.kh) * a.row_tiles + w.rt) * a.most * PG_WARPS + c * PG_WARPS + threadIdx.x / 32) *
                        part_floats(a.P, a.D);
}

// The outputs of a unit from its warps' (m, l, sums), or in a cluster from all
// blocks' of them, each block a part.  ms, ls [PG_WARPS][R]; os [PG_WARPS][R]
// [pitch]; spare: shared memory that no other block reads.
template <typename T>
__device__ __forceinline__ void join_warps(const PagedArgs& a, const float* ms, const float* ls, const float* os, int pitch,
                                           float* spare, const Work& w, int rows, int h0, int vis) {
    T* out = static_cast<T*>(a.o) + ((int64_t)w.b * a.H + h0) * a.D;
    const float nothing = vis < 0 ? __int_as_float(0x7fffffff) : 0.f;
    if (a.splits == 1) {
        for (int i = threadIdx.x; i < rows * a.D; i += PG_WARPS * 32) {
            const int r = i / a.D, d = i - r * a.D;
            float M[PG_WARPS], L[PG_WARPS], X[PG_WARPS];
#pragma unroll
            for (int x = 0; x < PG_WARPS; ++x) {
                M[x] = ms[x * a.R + r];
                L[x] = ls[x * a.R + r];
                X[x] = os[(x * a.R + r) * pitch + d];
            }
            out[i] = zg_from_float<T>(w.n == 0 ? nothing : Warps(M, L)(X));
        }
        return;
    }
    cluster_sync_all();
    // this thread's first output's sums, on their way while the factors are formed
    int i = (int)blockIdx.x % a.splits * PG_WARPS * 32 + threadIdx.x;
    float x[PG_WARPS][PG_CLUSTER];
    auto take = [&]() {
        if (i >= rows * a.D) return;
        const int r = i / a.D, d = i - r * a.D;
#pragma unroll
        for (int y = 0; y < PG_WARPS; ++y)
#pragma unroll
            for (int c = 0; c < PG_CLUSTER; ++c)
                if (c < w.n) x[y][c] = cluster_float(os + (y * a.R + r) * pitch + d, c);
    };
    take();
    // per row and warp: the factors of each block's chunk, and the end's maximum and sum
    float2* factor = reinterpret_cast<float2*>(spare);          // [R][PG_WARPS][PG_CLUSTER]
    float* end = spare + 2 * a.R * PG_WARPS * PG_CLUSTER;       // [R][PG_WARPS][2]
    if ((int)threadIdx.x < rows * PG_WARPS) {  // at most 64
        const int at = threadIdx.x, r = at / PG_WARPS, y = at % PG_WARPS;
        float m[PG_CLUSTER], l[PG_CLUSTER], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int c = 0; c < PG_CLUSTER; ++c)
            if (c < w.n) {
                m[c] = cluster_float(ms + y * a.R + r, c);
                l[c] = cluster_float(ls + y * a.R + r, c);
            }
#pragma unroll
        for (int c = 0; c < PG_CLUSTER; ++c)
            if (c < w.n) {
                const Fold fold(M, L, m[c], l[c]);
                factor[at * PG_CLUSTER + c] = make_float2(fold.before, fold.next);
            }
        end[2 * at] = M;
        end[2 * at + 1] = L;
    }
    __syncthreads();
    while (i < rows * a.D) {
        const int r = i / a.D;
        float M[PG_WARPS], L[PG_WARPS], X[PG_WARPS];
#pragma unroll
        for (int y = 0; y < PG_WARPS; ++y) {
            M[y] = end[2 * (r * PG_WARPS + y)];
            L[y] = end[2 * (r * PG_WARPS + y) + 1];
            X[y] = 0.f;
#pragma unroll
            for (int c = 0; c < PG_CLUSTER; ++c)
                if (c < w.n) {
                    const float2 f = factor[(r * PG_WARPS + y) * PG_CLUSTER + c];
                    X[y] = __fmaf_rn(x[y][c], f.y, __fmul_rn(X[y], f.x));
                }
        }
        out[i] = zg_from_float<T>(w.n == 0 ? nothing : Warps(M, L)(X));
        i += a.splits * PG_WARPS * 32;
        take();
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
// positions where a warp goes on after 16.  What costs is the instructions
// around them: with up to 8 heads (TALL not set) a lane's second row is none,
// and has no weights, sums or folds (64 sequences of 1000 to
// 4000: 84.7 -> 83.1 us; 250 of up to 250: 43 -> 39; 64 of up to 2000 at D = 256: 89 -> 80).
template <int DP, int STAGES, bool SHARE, bool TALL>
__global__ void __launch_bounds__(PG_WARPS * 32) paged_mma_kernel(const PagedArgs a) {
    using T = __nv_bfloat16;
    constexpr int CPR = DP / 8;             // 16-byte chunks of a row
    constexpr int TILE = 16 * DP * 2;       // bytes of 16 key (or value) rows
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float ms[PG_WARPS * 16], ls[PG_WARPS * 16];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    Work w = work_of<SHARE>(a);
    if (!w.on) return;
    const int b = w.b, kh = w.kh, rt = w.rt;
    const int rows = a.G - rt * 16 < 16 ? a.G - rt * 16 : 16;
    const int h0 = kh * a.G + rt * 16;
    const Seen see = seen_by(a, b);
    const bool whole = !SHARE && a.splits == 1;
    w.positions(a, see.vis, whole);
    const float lift = (float)lift_of(see.vis);
    const int c0 = w.first, end = w.end;  // this block: [c0, end)
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
                qf[k][e] = (TALL || e % 2 == 0) && r < rows && d < a.D ? *reinterpret_cast<const uint32_t*>(q + (int64_t)r * a.D + d) : 0u;
            }
    }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // rows lane/4 and lane/4 + 8, in units of log2

    const int k_row = (lane % 8) + 8 * (lane / 16), k_chunk = (lane / 8) % 2;
    const int v_row = (lane % 8) + 8 * ((lane / 8) % 2), v_chunk = lane / 16;
    // The chunks before this one.  With DP = 256 in shared memory: behind the
    // ring of three stages there is room for 8 rows, behind one of two for 16.
    static_assert(DP < 256 || SHARE || TALL == (STAGES == 2), "room for the chunks before");
    constexpr int ROWS = TALL ? 16 : 8;
    float M[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f};
    float kept[DP == 256 ? 1 : DP / 8][4];
    float* kept_far = reinterpret_cast<float*>(smem + PG_WARPS * STAGES * 2 * TILE) + warp * ROWS * DP + lane;
    auto so_far = [&](int d, int e) -> float& {
        if constexpr (DP == 256) return kept_far[(d * (ROWS / 4) + e) * 32];
        else return kept[d][e];
    };
    if constexpr (!SHARE) {
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
#pragma unroll
            for (int e = 0; e < ROWS / 4; ++e) so_far(d, e) = 0.f;
    }
    if (whole) w.chunks(a, see.vis, true);
    const int per_chunk = w.chunk / (16 * PG_WARPS);  // tiles of a chunk for each warp
    int i = 0;
    for (int c = w.c0; c < w.c1; ++c) {
        const int upto = (c + 1 - w.c0) * per_chunk < tiles ? (c + 1 - w.c0) * per_chunk : tiles;
#pragma unroll 1
        for (; i < upto; ++i) {
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
                for (int e = 0; e < ROWS / 4; ++e) {
                    s[j][e] = t0 + j * 8 + (lane % 4) * 2 + (e & 1) < end ? __fmul_rn(s[j][e], a.scale) : -INFINITY;
                    if (e < 2) n0 = fmaxf(n0, s[j][e]);
                    else n1 = fmaxf(n1, s[j][e]);
                }
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) {
                n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
                if (TALL) n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
            }
            n0 = fmaxf(n0, m0);
            n1 = fmaxf(n1, m1);
            const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
            const float b0l = b0 + lift, b1l = b1 + lift;
            if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
                const float f0 = exp2_fast(m0 - b0), f1 = exp2_fast(m1 - b1);
                l0 *= f0;
                l1 *= f1;
#pragma unroll
                for (int d = 0; d < DP / 8; ++d) {
                    o[d][0] *= f0;
                    o[d][1] *= f0;
                    if (TALL) {
                        o[d][2] *= f1;
                        o[d][3] *= f1;
                    }
                }
                m0 = n0;
                m1 = n1;
            }
            // weights, rounded to bf16 as the second product's operand (their sum
            // is of the unrounded ones): half a step of each weight, 2^-8
            uint32_t p[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float p0 = exp2_fast(s[j][0] - b0l), p1 = exp2_fast(s[j][1] - b0l);
                l0 += p0 + p1;
                p[2 * j] = pack_bf16(p0, p1);
                p[2 * j + 1] = 0u;
                if (TALL) {
                    const float p2 = exp2_fast(s[j][2] - b1l), p3 = exp2_fast(s[j][3] - b1l);
                    l1 += p2 + p3;
                    p[2 * j + 1] = pack_bf16(p2, p3);
                }
            }
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t f[4];
                ldmatrix4_t(f, vt + v_row * (DP * 2) + (((2 * d + v_chunk) ^ (v_row & 7)) * 16));
                mma_bf16(o[2 * d], p, f[0], f[1]);
                mma_bf16(o[2 * d + 1], p, f[2], f[3]);
            }
        }
        // this warp's leaf
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, x);
            if (TALL) l1 += __shfl_xor_sync(0xffffffffu, l1, x);
        }
        if constexpr (SHARE) {
            if (__any_sync(0xffffffffu, bad)) l0 = l1 = __int_as_float(0x7fffffff);
            float* leaf = leaf_of(a, w, c);
            const int pitch = pad4(a.D);
#pragma unroll
            for (int e = 0; e < ROWS / 8; ++e) {
                const int r = lane / 4 + 8 * e;
                if (r >= rows) continue;
#pragma unroll
                for (int d = 0; d < DP / 8; ++d)
                    if (d * 8 < a.D)
                        *reinterpret_cast<float2*>(leaf + r * pitch + d * 8 + (lane % 4) * 2) = make_float2(o[d][2 * e], o[d][2 * e + 1]);
                if (lane % 4 == 0) {
                    leaf[a.P * pitch + r] = e ? m1 : m0;
                    leaf[a.P * pitch + a.P + r] = e ? l1 : l0;
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < ROWS / 8; ++r) {
                const Fold fold(M[r], L[r], r ? m1 : m0, r ? l1 : l0);
#pragma unroll
                for (int d = 0; d < DP / 8; ++d)
#pragma unroll
                    for (int e = 2 * r; e < 2 * r + 2; ++e) so_far(d, e) = fold(so_far(d, e), o[d][e]);
            }
        }
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
#pragma unroll
            for (int e = 0; e < ROWS / 4; ++e) o[d][e] = 0.f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
    }
    copy_wait<0>();
    if constexpr (!SHARE) {
        bad = __syncthreads_or(bad);  // the rings are free from here on
        float* os = reinterpret_cast<float*>(smem);  // [PG_WARPS][16][DP]
        const int r = lane / 4;
        if (lane % 4 == 0) {
            ms[warp * 16 + r] = M[0];
            ls[warp * 16 + r] = bad ? __int_as_float(0x7fffffff) : L[0];
            if (TALL) {
                ms[warp * 16 + r + 8] = M[1];
                ls[warp * 16 + r + 8] = bad ? __int_as_float(0x7fffffff) : L[1];
            }
        }
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
            float* to = os + (warp * 16 + r) * DP + d * 8 + (lane % 4) * 2;
            *reinterpret_cast<float2*>(to) = make_float2(so_far(d, 0), so_far(d, 1));
            if (TALL) *reinterpret_cast<float2*>(to + 8 * DP) = make_float2(so_far(d, 2), so_far(d, 3));
        }
        __syncthreads();
        join_warps<T>(a, ms, ls, os, DP, os + PG_WARPS * 16 * DP, w, rows, h0, see.vis);
    }
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
    Work w = work_of<SHARE>(a);
    if (!w.on) return;
    const int b = w.b, kh = w.kh, rt = w.rt;
    const int rows = a.G - rt * GT < GT ? a.G - rt * GT : GT;
    const int h0 = kh * a.G + rt * GT;
    const Seen see = seen_by(a, b);
    const bool whole = !SHARE && a.splits == 1;
    w.positions(a, see.vis, whole);
    const float low = ldexpf(1.f, -lift_of(see.vis));
    const int c0 = w.first, end = w.end;
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
    float kept[GT][NI], M[GT], L[GT];  // the chunks before this one
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        M[g] = -INFINITY;
        L[g] = 0.f;
#pragma unroll
        for (int x = 0; x < NI; ++x) kept[g][x] = 0.f;
    }
    if (whole) w.chunks(a, see.vis, true);
    const int per_chunk = w.chunk / (TT * PG_WARPS);
    int i = 0;
    for (int c = w.c0; c < w.c1; ++c) {
        const int upto = (c + 1 - w.c0) * per_chunk < tiles ? (c + 1 - w.c0) * per_chunk : tiles;
#pragma unroll 1
        for (; i < upto; ++i) {
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
                s[g] = exp2f(s[g] - base) * low;
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
        // this warp's leaf
#pragma unroll
        for (int g = 0; g < GT; ++g)
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], x);
        if constexpr (SHARE) {
            const bool spoilt = __any_sync(0xffffffffu, bad);
            float* leaf = leaf_of(a, w, c);
            const int pitch = pad4(a.D);
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                if (g >= rows) continue;
#pragma unroll
                for (int x = 0; x < NI; ++x)
                    if (lane + 32 * x < pitch) leaf[g * pitch + lane + 32 * x] = o[g][x];
                if (lane == 0) {
                    leaf[a.P * pitch + g] = m[g];
                    leaf[a.P * pitch + a.P + g] = spoilt ? __int_as_float(0x7fffffff) : l[g];
                }
            }
        } else {
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const Fold fold(M[g], L[g], m[g], l[g]);
#pragma unroll
                for (int x = 0; x < NI; ++x) kept[g][x] = fold(kept[g][x], o[g][x]);
            }
        }
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int x = 0; x < NI; ++x) o[g][x] = 0.f;
        }
    }
    copy_wait<0>();
    if constexpr (!SHARE) {
        bad = __syncthreads_or(bad);
        float* os = reinterpret_cast<float*>(smem);  // [PG_WARPS][GT][DMAX]
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            if (lane == 0) {
                ms[warp * GT + g] = M[g];
                ls[warp * GT + g] = bad ? __int_as_float(0x7fffffff) : L[g];
            }
#pragma unroll
            for (int x = 0; x < NI; ++x) os[(warp * GT + g) * DMAX + lane + 32 * x] = kept[g][x];
        }
        __syncthreads();
        join_warps<T>(a, ms, ls, os, DMAX, os + PG_WARPS * GT * DMAX, w, rows, h0, see.vis);
    }
}

// Folds the chunks of one query head in their order, each warp's apart, and
// joins those: a block per (b, h) and 32 columns, a warp for each warp of the
// chunks' blocks, a lane a column.  The factors come of the maxima alone; they
// are formed first, while the first sums are on their way.  It is launched so
// that its blocks start as the last chunk's block ends.  (With its blocks
// waiting in their places meanwhile, one sequence of 131000 took 54.3 us
// instead of 51.6.)
constexpr int PJ_MOST = 448, PJ_AHEAD = 32;
template <typename T>
__global__ void __launch_bounds__(PG_WARPS * 32) paged_join_kernel(const PagedArgs a) {
    __shared__ float2 factor[PG_WARPS][PJ_MOST];
    __shared__ float ls[PG_WARPS][PJ_MOST], Xs[PG_WARPS][32], Ms[PG_WARPS], Ls[PG_WARPS];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int b = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x % a.H), d = (int)blockIdx.y * 32 + lane;
    const int kh = h / a.G, rt = h % a.G / a.R, r = h % a.G % a.R;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched before the chunks' kernel has ended
    const int vis = seen_by(a, b).vis, n = chunks_of(a, vis);
    const int64_t pf = part_floats(a.P, a.D), step = PG_WARPS * pf;
    const int pitch = pad4(a.D);
    const float* part = a.part + ((((int64_t)b * a.K + kh) * a.row_tiles + rt) * a.most * PG_WARPS + warp) * pf;
    const float* column = part + r * pitch + (d < pitch ? d : 0);
    float x[PJ_AHEAD];
    auto load = [&](int c0) {
#pragma unroll
        for (int e = 0; e < PJ_AHEAD; ++e)
            if (c0 + e < n) x[e] = column[(c0 + e) * step];
    };
    load(0);
    float M = -INFINITY;  // of the chunks before these 32
    for (int c0 = 0; c0 < n; c0 += 32) {
        const float* ml = part + (c0 + lane) * step + a.P * pitch;
        const bool on = c0 + lane < n;
        const float m = on ? ml[r] : -INFINITY;
        if (on) ls[warp][c0 + lane] = ml[a.P + r];
        float top = m;  // of these up to this lane's
#pragma unroll
        for (int f = 1; f < 32; f <<= 1) {
            const float y = __shfl_up_sync(0xffffffffu, top, f);
            if (lane >= f) top = fmaxf(top, y);
        }
        const float above = __shfl_up_sync(0xffffffffu, top, 1);
        float before = lane ? fmaxf(M, above) : M, sum = 0.f;
        const Fold fold(before, sum, m, 0.f);
        if (on) factor[warp][c0 + lane] = make_float2(fold.before, fold.next);
        M = fmaxf(M, __shfl_sync(0xffffffffu, top, 31));
    }
    __syncwarp();
    float X = 0.f, L = 0.f;
    for (int c0 = 0; c0 < n; c0 += PJ_AHEAD) {
#pragma unroll
        for (int e = 0; e < PJ_AHEAD; ++e)
            if (c0 + e < n) {
                const float2 f = factor[warp][c0 + e];
                X = __fmaf_rn(x[e], f.y, __fmul_rn(X, f.x));
                L = __fmaf_rn(ls[warp][c0 + e], f.y, __fmul_rn(L, f.x));
            }
        if (c0 + PJ_AHEAD < n) load(c0 + PJ_AHEAD);
    }
    Xs[warp][lane] = X;
    if (lane == 0) {
        Ms[warp] = M;
        Ls[warp] = L;
    }
    __syncthreads();
    if (warp || d >= a.D) return;
    float Mw[PG_WARPS], Lw[PG_WARPS], Xw[PG_WARPS];
#pragma unroll
    for (int w = 0; w < PG_WARPS; ++w) {
        Mw[w] = Ms[w];
        Lw[w] = Ls[w];
        Xw[w] = Xs[w][lane];
    }
    const float out = vis < 0 ? __int_as_float(0x7fffffff) : n == 0 ? 0.f : Warps(Mw, Lw)(Xw);
    static_cast<T*>(a.o)[((int64_t)b * a.H + h) * a.D + d] = zg_from_float<T>(out);
}

// How a call is cut: R query rows of a unit, the chunks of a sequence, and
// what the blocks are.
struct PagedPlan {
    int R, row_tiles, P, each, most, splits, share;
    bool mma, leaves;  // leaves: in the workspace
};

PagedPlan paged_plan(int64_t B, int H, int K, int D, int64_t longest, int window, int sinks, int dtype) {
    PagedPlan p{};
    const int G = H / K;
    p.mma = dtype == ZG_BF16 && D % 8 == 0;
    p.R = p.mma ? 16 : G == 1 ? 1 : G <= 4 ? 4 : 8;
    p.row_tiles = (G + p.R - 1) / p.R;
    p.P = G < p.R ? G : p.R;
    int64_t vis = longest;
    if (window > 0 && (int64_t)window + sinks < vis) vis = (int64_t)window + sinks;
    // Blocks that run on an SM at once, by the instances' shared memory and
    // registers: of the tensor cores' two, above 128 columns (192 KB) one; of
    // the FMA path three, above 128 columns (up to 255 registers) two.
    const int per_sm = p.mma ? (D <= 128 ? 2 : 1) : D <= 128 ? 3 : 2;
    // A sequence alone fills the places of a whole chip once (148 SMs: a
    // constant, as the cut is part of the result).
    const int heads = K * p.row_tiles;
    p.each = per_sm * 148 / heads > 1 ? per_sm * 148 / heads : 1;
    const int64_t fill = (vis + PG_CHUNK - 1) / PG_CHUNK;
    p.most = (int)(fill < p.each ? (fill > 0 ? fill : 1) : p.each);
    // Units that fill most places are not cut further, nor short ones that fill
    // half of them (32 sequences of up to 1000, 32 heads of 8 key heads: 27.3
    // us, 41.6 with leaves in the workspace).  A block of its own for each chunk
    // costs its pipeline's filling: 64 sequences of different lengths cut four
    // times as often were 126 us.  Below that a cluster of up to eight chunks
    // joins them by itself.  Otherwise the leaves go through the workspace: with
    // two, four or eight equal parts of a unit (16 sequences of up to 8000, 8 key
    // heads: 71.6 us, by the lengths 76.7), or where that would not fill the
    // places, shared out by the lengths that the device knows (by the table's
    // width a sequence of 8000 in a table of 131072 took 42 us, now 11.9).
    const int64_t units = B * heads, places = (int64_t)per_sm * zg::sm_count();
    p.splits = 1;
    if (5 * units >= 4 * places || (2 * units >= places && p.most <= 8) || p.most == 1) return p;
    const int blocks = p.most <= 2 ? 2 : p.most <= 4 ? 4 : 8;
    const int64_t parts = (places + units - 1) / units;
    if (p.most <= PG_CLUSTER && units * blocks <= 2 * places) {
        p.splits = blocks;
    } else {
        p.leaves = true;
        if (parts <= 8)
            p.splits = parts <= 2 ? 2 : parts <= 4 ? 4 : 8;
        else
            p.share = (int)places;  // more than eight times the units, of which there are less than 64
    }
    return p;
}

size_t paged_workspace(const PagedPlan& p, int64_t B, int K, int D) {
    return p.leaves ? (size_t)(B * K * p.row_tiles * p.most * PG_WARPS * part_floats(p.P, D)) * sizeof(float) : 0;
}

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
    c.numAttrs = a.splits > 1 && !a.part ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&c, f, args...);
    if (e != cudaSuccess) return zg::fail(ZG_ERR_CUDA, "zg_paged_attention: %s", cudaGetErrorString(e));
    return zg::check_launch("zg_paged_attention");
}

// STAGES of the ring, OWN of those of a kernel that keeps its chunks' sums.
template <int DP, int STAGES, int OWN, bool TALL>
int launch_mma(const PagedArgs& a, int64_t blocks, cudaStream_t st) {
    const size_t smem = (size_t)PG_WARPS * (a.part ? STAGES : OWN) * 2 * 16 * DP * 2 +
                        (DP == 256 && !a.part ? PG_WARPS * (TALL ? 16 : 8) * DP * sizeof(float) : 0);
    const auto f = a.part ? paged_mma_kernel<DP, STAGES, true, TALL> : paged_mma_kernel<DP, OWN, false, TALL>;
    if (int rc = set_smem(f, smem)) return rc;
    zg::LaunchTimer zg_lt_("paged_attention", st);
    return launch_split(f, a, blocks, smem, st, a);
}
template <bool TALL>
int launch_mma_any(const PagedArgs& a, int64_t blocks, cudaStream_t st) {
    return a.D <= 64    ? launch_mma<64, 4, 4, TALL>(a, blocks, st)
           : a.D <= 128 ? launch_mma<128, 3, 3, TALL>(a, blocks, st) : launch_mma<256, 3, TALL ? 2 : 3, TALL>(a, blocks, st);
}

template <typename T, int PARTS, int GT>
int launch_fma(const PagedArgs& a, int vec, int64_t blocks, cudaStream_t st) {
    const size_t ring = (size_t)PG_WARPS * PG_FMA_STAGES * 2 * (32 / PARTS) * (32 * PARTS * sizeof(T) + 16);
    // behind the end's sums there is room for a cluster's factors
    const size_t out = (size_t)PG_WARPS * GT * (32 * PARTS + 2 * PG_CLUSTER + 2) * sizeof(float);
    const size_t smem = ring > out ? ring : out;
    const auto f = a.part ? paged_fma_kernel<T, PARTS, GT, true> : paged_fma_kernel<T, PARTS, GT, false>;
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
    return paged_workspace(paged_plan(B, H, K, D, (int64_t)max_pages * page, window, sinks, dtype), B, K, D);
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
    const size_t need = paged_workspace(p, B, K, D);
    if (need && (!workspace || workspace_bytes < need))
        return zg::fail(ZG_ERR_WORKSPACE, "zg_paged_attention: workspace of %zu bytes needed", need);
    const int64_t blocks = p.share ? p.share : B * K * p.row_tiles * p.splits;
    if (blocks > INT32_MAX) return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: too many rows");
    const int n = 16 / (int)zg::dtype_size(dtype);
    const int vec = D % n == 0 && aligned16(k_pages) && aligned16(v_pages);
    PagedArgs a{q, k_pages, v_pages, table, lengths, o, p.leaves ? static_cast<float*>(workspace) : nullptr, ldq, n_pages, page, max_pages,
                (int)B, H, K, D, H / K, p.row_tiles, p.R, p.P, window, sinks, p.splits, p.share, p.each, p.most, p.mma ? 2 * PG_CHUNK : PG_CHUNK,
                (float)(1.4426950408889634 / sqrt((double)D))};
    cudaStream_t st = zg::as_stream(stream);
    int rc;
    if (p.mma && vec && ldq % 2 == 0 && (reinterpret_cast<uintptr_t>(q) & 3) == 0) {
        rc = p.P > 8 ? launch_mma_any<true>(a, blocks, st) : launch_mma_any<false>(a, blocks, st);
    } else if (p.mma) {
        return zg::fail(ZG_ERR_INVALID, "zg_paged_attention: bf16 pages with D a multiple of 8 must be 16-byte "
                                        "aligned, q 4-byte aligned with an even pitch");
    } else {
        rc = dtype == ZG_BF16 ? launch_fma_any<__nv_bfloat16>(a, vec, blocks, st)
                              : launch_fma_any<float>(a, vec, blocks, st);
    }
    if (rc != ZG_OK || !p.leaves) return rc;
    zg::LaunchTimer zg_lt_("paged_join", st);
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(B * H), (unsigned)((D + 31) / 32));
    c.blockDim = dim3(PG_WARPS * 32);
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
