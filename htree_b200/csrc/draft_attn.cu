// Attention of drafted tokens over a paged cache and over the drafts that lead to them.
//
//     s_ij = scale * q_i . k_j,   lse_i = log sum_j e^s_ij,   out_i = sum_j e^(s_ij - lse_i) v_j      over the cached j and i's line of drafts
//
// in one pass over the keys: with a reference r for each row, mass = sum 2^(s' - r) and the sums of 2^(s' - r) v_j, s' = s log2 e, and both
// scaled when r moves.
//
// Work: the query rows that share a key/value head (drafts x heads of the group) are cut into row tiles; a unit is a request, a key/value
// head and a row tile, and its keys are tiles: the cached tokens first, then the drafts.  All tiles of all units stand in one line that is
// cut into equal parts, one per block, whatever the lengths (which only the device knows).  A unit that lies in one part is finished
// there; of the others every part leaves its unnormalised sum, its reference and its mass, which a second kernel joins in the order of the
// parts: the result does not depend on timing.
#include "cache.cuh"
#include "mma_common.cuh"

#include <cuda.h>

namespace htree {

constexpr int kMaxTree = 1024;
constexpr int64_t kMaxLength = int64_t(1) << 30;
constexpr int kSlice = 16, kTile = 64;    // keys of a tile: slices, FFMA

struct DraftParams {
    const char* q;
    const char* k;
    const char* v;
    const char* ck;
    const char* cv;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* parents;
    void* out;
    float* lse;
    float* part;              // per slot: rows x V sums, then rows x {reference, mass}; slots 2c and 2c+1 are part c's first and last unit
    int4* tasks;              // what there is to join: per unit, or per part where there are more units than parts (see Task)
    int32_t* status;
    int64_t q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h;                  // strides in bytes
    int64_t ck_page, ck_row, ck_h, cv_page, cv_row, cv_h;
    int64_t table_stride;
    int32_t B, N, H, Hkv, G, K, V, pages;
    int32_t rows, row_tiles, shift, draft_tiles;                           // rows of a row tile, log2 of the keys of a tile
    int32_t room;             // tokens that a row of the table can name
    int32_t whole;            // short tables: parts of whole units, and nothing to join
    int32_t grid, least, by_unit, team;                                    // parts at most; tiles of a part at least; how tasks are indexed, and joined
    int32_t variant;          // which kernel (choose)
    int32_t boxes;            // tcgen05 kernel: what comes by tensor maps: 1 pages of whole slices of sixteen tokens, 2 q, 4 drafts
    int32_t box_rows;         // tokens of a box of a whole tile: as many as pages allow, up to the tile
    int32_t neg;              // tensor-core kernels: the scale is negative, c its magnitude and q's signs are turned
    float c;                  // scale * log2 e
    FastDiv page, group, per_head;      // by the page size, by G, by row_tiles
};

// ---- the line of tiles -------------------------------------------------------------------------------------------------------

__device__ __forceinline__ int draft_length(const DraftParams& p, int b, bool* bad) {
    const int len = p.lengths[b], in = min(max(len, 0), p.room);
    if (in != len) *bad = true;
    return in;
}
__device__ __forceinline__ int tiles_for(const DraftParams& p, int len) { return ((len + (1 << p.shift) - 1) >> p.shift) + p.draft_tiles; }
__device__ __forceinline__ int draft_tiles_of(const DraftParams& p, int b) {
    bool dull = false;
    return tiles_for(p, draft_length(p, b, &dull));
}

// Where a part of the line is: request, unit of the request (head * row_tiles + row tile), tile of the unit.
struct Place {
    int b, unit, tile, tiles, len;
    __device__ __forceinline__ void enter(const DraftParams& p, int b_) {
        bool dull = false;
        b = b_;
        len = draft_length(p, b, &dull);
        tiles = tiles_for(p, len);
    }
    __device__ __forceinline__ void next(const DraftParams& p) {
        if (++tile < tiles) return;
        tile = 0;
        if (++unit < p.Hkv * p.row_tiles) return;
        unit = 0;
        if (b + 1 < p.B) enter(p, b + 1);
    }
};

// The line and its parts, in 32 bits where it fits them (a 64-bit division takes as long as a load): the first `more` parts have each + 1
// tiles, the others `each`.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) { return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }
struct Line {
    int64_t all, each, more;
    int parts;
    Line() = default;
    __device__ __forceinline__ Line(const DraftParams& p, int64_t all_) : all(all_) {
        parts = all >= (int64_t)p.grid * p.least ? p.grid : (int)(((uint32_t)all + p.least - 1) / (uint32_t)p.least);
        each = divide(all, parts);
        more = all - each * parts;
    }
    __device__ __forceinline__ int64_t start(int64_t c) const { return c * each + (c < more ? c : more); }
    __device__ __forceinline__ int part_of(int64_t x) const {
        const int64_t big = more * (each + 1);
        return (int)(x < big ? divide(x, each + 1) : more + divide(x - big, each));
    }
};

// The line, and the place where this block's part starts (x0; it ends before x1).  False for a block without a part.  Every thread takes a
// stretch of requests: of a warp's where there are few, so that no warp waits for another, of the block's where there are many.
__device__ __forceinline__ uint32_t scan_tiles(const DraftParams& p, int me, int threads, uint32_t& mine, uint32_t& before, int& b0) {
    const int per = threads == 32 ? (p.B + 31) >> 5 : (p.B + threads - 1) / threads, b1 = min(me * per + per, p.B);
    b0 = min(me * per, p.B);
    mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) mine += (uint32_t)draft_tiles_of(p, b);
    uint32_t in = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, in, o);
        if ((me & 31) >= o) in += y;
    }
    before = in - mine;
    return __shfl_sync(0xffffffffu, in, 31);
}
// (The tiles of all requests for one unit are below 2^31, which the launch has checked; those of all units need not be.)
template <int NT>
__device__ __forceinline__ bool find_part(const DraftParams& p, Place& at, Line& line, int64_t& x0, int64_t& x1) {
    __shared__ uint32_t scratch[NT / 32], found[2];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, units = p.Hkv * p.row_tiles;
    if (p.whole) {
        const int64_t all = (int64_t)p.B * units, u0 = divide(blockIdx.x * all, p.grid), u1 = divide((blockIdx.x + 1) * all, p.grid);
        if (u0 == u1) return false;
        const int b0 = (int)divide(u0, units);
        x0 = x1 = 0;
        for (int64_t u = u0, b = b0; u < u1; ++b) {              // units of request b
            const int64_t to = min((b + 1) * units, u1);
            x1 += (to - u) * draft_tiles_of(p, (int)b);
            u = to;
        }
        at.enter(p, b0);
        at.unit = (int)(u0 - (int64_t)b0 * units);
        at.tile = 0;
        return true;
    }
    const bool few = p.B <= 128;
    uint32_t mine, before;
    int b0;
    uint32_t all = scan_tiles(p, few ? lane : tid, few ? 32 : NT, mine, before, b0);
    if (!few) {
        if (lane == 0) scratch[w] = all;
        __syncthreads();
        all = 0;
#pragma unroll 1
        for (int i = 0; i < NT / 32; ++i) {
            if (i < w) before += scratch[i];
            all += scratch[i];
        }
    }
    line = Line(p, (int64_t)all * units);
    if ((int)blockIdx.x >= line.parts) return false;
    x0 = line.start(blockIdx.x);
    x1 = line.start(blockIdx.x + 1);
    const uint32_t want = (uint32_t)divide(x0, units);               // which tile of the requests, were there one unit each
    const bool here = want >= before && want < before + mine;
    int b = b0;
    if (here)
#pragma unroll 1
        for (uint32_t t = draft_tiles_of(p, b); want >= before + t; t = draft_tiles_of(p, ++b)) before += t;
    if (few) {
        const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
        b = __shfl_sync(0xffffffffu, b, from);
        before = __shfl_sync(0xffffffffu, before, from);
    } else {
        if (here) { found[0] = (uint32_t)b; found[1] = before; }
        __syncthreads();
        b = (int)found[0];
        before = found[1];
    }
    at.enter(p, b);
    const int64_t in = x0 - (int64_t)before * units;
    at.unit = (int)divide(in, at.tiles);
    at.tile = (int)(in - (int64_t)at.unit * at.tiles);
    return true;
}

// What there is to join of the unit that starts with tile u0 of the line, in part c: x = its request (-1: nothing), y = the unit of the
// request, z = part c, w = 2 * parts + (another unit came before it in part c).
__device__ __forceinline__ void leave_task(const DraftParams& p, const Place& at, int64_t u0, int64_t x0, int c, const Line& line, bool whole) {
    if (p.whole) return;
    int4 t = make_int4(-1, 0, 0, 0);
    if (!whole) t = make_int4(at.b, at.unit, c, 2 * (line.part_of(u0 + at.tiles - 1) - c + 1) + (x0 < u0 ? 1 : 0));
    if (p.by_unit) p.tasks[(int64_t)at.b * p.Hkv * p.row_tiles + at.unit] = t;
    else if (!whole) p.tasks[c] = t;
}

__device__ __forceinline__ int head_of(const DraftParams& p, int unit) { return (int)p.per_head.div((uint32_t)unit); }     // key/value head
// Row r of a row tile: draft and head.  False behind the last row.
__device__ __forceinline__ bool row_of(const DraftParams& p, int unit, int r, int& n, int& h) {
    const int kv = head_of(p, unit), row = (unit - kv * p.row_tiles) * p.rows + r;
    n = (int)p.group.div((uint32_t)row);
    h = kv * p.G + row - n * p.G;
    return row < p.N * p.G;
}

// Which of the drafts tile0 .. tile0 + 64 * W - 1 draft n reads.
template <int W>
__device__ __forceinline__ void draft_masks(const DraftParams& p, int b, int n, int tile0, uint64_t (&m)[W], bool* bad) {
    if (!p.parents) {                                        // a chain: n and all before it
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int upto = n - tile0 - 64 * i;
            m[i] = upto < 0 ? 0ull : upto >= 63 ? ~0ull : (2ull << upto) - 1ull;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) m[i] = 0;
    const int32_t* par = p.parents + (int64_t)b * p.N;
    // Parents come before their children: at most n steps, each as long as its load.  (With a branch on `up` in front of the bits, which then
    // waited for the load, a chain of 1024 given as a tree took 1010 us instead of 681.)
    for (int i = n; i >= tile0;) {
        const int up = par[i];
        const uint64_t bit = up < -1 ? 0ull : 1ull << ((i - tile0) & 63);            // (below -1: no draft, and the walk ends)
#pragma unroll
        for (int j = 0; j < W; ++j) m[j] |= (i - tile0) >> 6 == j ? bit : 0ull;
        *bad |= up >= i;
        i = up >= i ? -1 : up;
    }
}
__device__ __forceinline__ uint64_t draft_mask(const DraftParams& p, int b, int n, int tile0, bool* bad) {
    uint64_t m[1];
    draft_masks(p, b, n, tile0, m, bad);
    return m[0];
}
__device__ __forceinline__ bool is_draft(const DraftParams& p, int b, int n) { return !p.parents || p.parents[(int64_t)b * p.N + n] >= -1; }

// Where the row of key j of a tile starts (keys, values); false for what the tile does not have.
__device__ __forceinline__ bool key_row(const DraftParams& p, const Place& at, int kv, int j, const char*& k, const char*& v, bool* bad) {
    const int cached = at.tiles - p.draft_tiles;
    if (at.tile < cached) {
        const int pos = (at.tile << p.shift) + j;
        if (pos >= at.len) return false;
        const uint32_t i = p.page.div((uint32_t)pos);
        const int pg = __ldg(p.table + (int64_t)at.b * p.table_stride + i);
        if (pg < 0 || pg >= p.pages) { *bad = true; return false; }
        const int64_t in = (int64_t)(pos - i * p.page.d);
        k = p.ck + pg * p.ck_page + in * p.ck_row + kv * p.ck_h;
        v = p.cv + pg * p.cv_page + in * p.cv_row + kv * p.cv_h;
        return true;
    }
    const int n = ((at.tile - cached) << p.shift) + j;
    if (n >= p.N || !is_draft(p, at.b, n)) return false;
    k = p.k + at.b * p.k_b + n * p.k_n + kv * p.k_h;
    v = p.v + at.b * p.v_b + n * p.v_n + kv * p.v_h;
    return true;
}

// out and lse of a row from its sums (m in units of log2, as everywhere in the kernels); rows of drafts that are none are empty.
__device__ __forceinline__ float finish_scale(float mass) { return mass > 0.f ? 1.f / mass : (mass == 0.f ? 0.f : mass); }   // NaN stays NaN
__device__ __forceinline__ float finish_lse(float m, float mass) {
    return mass == 0.f ? -INFINITY : (m + log2f(mass)) * 0.69314718055994531f;
}

// ---- few query rows, and rows wider than 128: slices of keys ------------------------------------------------------------------

// HBM bounds these (fp32 with more than 4 rows: the FMA pipes, at 11 to 15 TFLOP/s); the products only have to keep up: mma.sync in 16
// bits, FFMA in fp32.  Measured, 32 requests, 8 heads of the cache, 4 query heads each: 16384 tokens of 128 in 359 us in bf16 (6.0 TB/s)
// and 762 in fp32 (5.6), of 64 in 213 and 413 (5.0 and 5.2), 8192 of 256 in 361 to 374 and 927 (5.8 and 4.6).  A tile is 16 keys and belongs to one warp, with a softmax of its own (reference,
// mass and sums in registers) and a ring of its own in shared memory that the warp fills by cp.async: the warps of a block do not wait for
// one another until the unit ends.  The line is cut into parts of whole blocks; the tiles of a part go round the block's warps.
// (One bulk copy of 256 bytes per lane and row instead: the compiler issues them lane by lane, 790 instructions a tile.)
//
// The reference of a row is not its running maximum but within kLag of it (powers of two that P may grow by before the sums are
// rescaled), so almost every tile needs one vote and no shuffles.  P is rounded to the type, half a step each; for fp16 the reference
// lies kBias below the maximum, so that weights down to 2^-22 of the largest keep all their digits and the largest stays below 2^15.
template <typename T> constexpr float kLag = 8.f;
template <> constexpr float kLag<__half> = 7.f;
template <typename T> constexpr float kBias = 0.f;
template <> constexpr float kBias<__half> = 8.f;

template <typename T> constexpr uint32_t kExpMask = 0x7f80u;
template <> constexpr uint32_t kExpMask<__half> = 0x7c00u;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// Values of drafts that are not finite must not meet the zero weights of the rows that do not read them: they are taken out of the tile
// (their rows noted) and added to the rows that do.  `piece`: 16 bytes in shared memory.  True if it held any.
template <typename T>
__device__ __forceinline__ bool take_out(uint32_t piece) {
    uint32_t u[4];
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(piece) : "memory");
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool lo = (u[i] & kExpMask<T>) == kExpMask<T>, hi = (u[i] >> 16 & kExpMask<T>) == kExpMask<T>;
        any |= lo | hi;
        u[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    }
    if (any) asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(piece), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
    return any;
}
// ... and what such a value adds to a row that reads it
template <typename T>
__device__ __forceinline__ float put_back(float o, const char* v, int col) {
    const float x = to_f<T>(reinterpret_cast<const T*>(v)[col]);
    return fabsf(x) <= 3.4028234e38f ? o : o + x;
}

template <typename T, int DK, int DV, int R> struct SliceShape {          // R query rows
    static constexpr bool f32 = sizeof(T) == 4;
    static constexpr int warps = DK + DV > 256 ? (f32 ? 3 : 6) : R == 32 ? 8 : f32 && DK + DV > 192 ? 6 : f32 && DK + DV > 128 ? 8 : 12;
    static constexpr int threads = warps * 32, rows = R;
    static constexpr int krow = DK * (int)sizeof(T) + 16, vrow = DV * (int)sizeof(T) + 16;             // 16 bytes more than a row: eight rows meet in no bank
    static constexpr int stage = kSlice * (krow + vrow);
    // columns of a joining round: what fits into the stage that the unit's last tile has left
    static constexpr int cols = f32 ? DV : DV == 128 && rows * 132 * 4 <= stage ? 128 : rows * 68 * 4 <= stage ? 64 : 32, jrow = cols + 4;
    static_assert(rows * jrow * 4 <= stage, "");
    static constexpr int weights = f32 ? warps * rows * kSlice * 4 : 0;
    static constexpr int fixed = 2 * warps * rows * 4 + (rows + 16) * 4 + rows * krow + weights;
    static constexpr int fit = (232448 - 512 - fixed) / (warps * stage);
    static constexpr int stages = fit > 4 ? 4 : fit;
    static_assert(stages >= 2, "");
    static constexpr int wm = 0, wl = wm + warps * rows * 4, sums = wl + warps * rows * 4, q = sums + (rows + 16) * 4, p = q + rows * krow,
                         ring = (p + weights + 127) / 128 * 128, total = ring + warps * stages * stage;
};

// The code of a part runs few times over (a handful of tiles, one or two joins), and instructions that run for the first time come at 8 to
// 10 cycles each: one loop, in which fetching, computing and joining stand once each, nothing unrolled that need not be.  (Unrolled, with
// the prologue and every refill inlined, a call of 1024 cached tokens took 38,000 cycles, 26,000 of them outside the tiles.)
template <typename T, int DK, int DV, int ROWS>
__global__ void __launch_bounds__(SliceShape<T, DK, DV, ROWS>::threads, 1) draft_slice_kernel(const __grid_constant__ DraftParams p) {
    using S = SliceShape<T, DK, DV, ROWS>;
    constexpr bool F32 = S::f32;
    constexpr int NT = S::threads, NW = S::warps, ST = S::stages, RM = F32 ? 1 : ROWS / 16, E = 16 / (int)sizeof(T);       // E: elements of 16 bytes
    extern __shared__ __align__(128) unsigned char sm[];
    float* wm = reinterpret_cast<float*>(sm + S::wm);
    float* wl = reinterpret_cast<float*>(sm + S::wl);
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, r4 = lane & 3;
    float* scale_of = reinterpret_cast<float*>(sm + S::sums);
    int* stage_of = reinterpret_cast<int*>(sm + S::sums) + ROWS;
    unsigned char* ring = sm + S::ring + w * ST * S::stage;
    const uint32_t ring_u = smem_u32(ring), q_u = smem_u32(sm + S::q);
    if (p.K < DK || p.V < DV) {        // columns that no copy writes
        for (int i = lane; i < ST * S::stage / 16; i += 32) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < ROWS * S::krow / 16; i += NT) reinterpret_cast<uint4*>(sm + S::q)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    chain_enter();
    Place at;
    Line line;
    int64_t x0, x1;
    if (tid == 0 && !p.by_unit && !p.whole) p.tasks[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (!find_part<NT>(p, at, line, x0, x1)) return;
    const int n_tiles = (int)(x1 - x0);
    bool bad = false;
    { bool b = false; draft_length(p, at.b, &b); bad |= b; }

    // The rows of q of a unit, to shared memory.
    auto fetch_q = [&](const Place& pl) {
#pragma unroll 1
        for (int i = tid; i < ROWS * (DK / E); i += NT) {
            const int r = i / (DK / E), c = i % (DK / E);
            int n, h;
            const bool on = row_of(p, pl.unit, r, n, h);
            if (c * E < p.K) cp_async16_or_zero(q_u + r * S::krow + c * 16, on ? p.q + pl.b * p.q_b + n * p.q_n + h * p.q_h + c * 16 : p.q, on);
        }
    };
    fetch_q(at);

    // This warp's tiles are w, w + NW, ...  `ahead` is the next one to fetch; lane j (and j + 16) knows the page of its key j, read one fetch
    // before it is needed.
    Place ahead = at;
    auto look = [&](const Place& pl) {
        const int pos = pl.tile * kSlice + (lane & 15);
        return pl.tile < pl.tiles - p.draft_tiles && pos < pl.len ? __ldg(p.table + (int64_t)pl.b * p.table_stride + p.page.div((uint32_t)pos)) : -1;
    };
    constexpr int KP = DK > 32 * E ? DK / (32 * E) : 1, VP = DV > 32 * E ? DV / (32 * E) : 1;                 // pieces of a row of a lane,
    constexpr int KL = DK / E / KP, VL = DV / E / VP;                                                         // 32 apart; lanes of a row
    const uint32_t kdst = ring_u + lane / KL * S::krow + lane % KL * 16, vdst = ring_u + kSlice * S::krow + lane / VL * S::vrow + lane % VL * 16;
    auto kcol = [&](int h) { return (lane % KL + 32 * h) * E < p.K; };
    auto vcol = [&](int h) { return (lane % VL + 32 * h) * E < p.V; };
    const int64_t kstep = p.ck_row * (32 / KL), vstep = p.cv_row * (32 / VL);
    uint64_t keys_of = 0;                  // which keys a stage has: 16 bits each

    // 16 bits: fragments of RM x 16 rows, this thread's rows g and g + 8 of each; fp32: all rows' columns CW * lane .., and this lane's keys' mass
    constexpr int CW = DV / 32;
    float o[RM][DV / 8][4], ref[RM][2], mass[RM][2], fo[F32 ? ROWS : 1][CW], fref[F32 ? ROWS : 1], fmass[F32 ? ROWS : 1];
    uint32_t qf[RM][DK / 16][4];
    int piece = 0, first = 0, end = 0;     // tiles first .. end of the part: the share of the present unit
    int had = -1;                          // the stage of this warp's last tile of the unit, or -1: it had none
    bool first_piece = true, q_ready = false;
    int step = w;                          // how far `ahead` has to go before the next fetch
    int page_next = -1;
    for (int k = 0;; ++k) {
        const int t = k - (ST - 1), mine = w + t * NW;   // the tile to compute in this round
        while (t >= 0 && mine >= end) {
            if (piece > 0) {
                // the block's warps, those that had a tile of the unit: one reference, the sums added, through the stages that they have left
                if (had >= 0) {
                    if constexpr (F32) {
#pragma unroll
                        for (int r = 0; r < ROWS; ++r) {
                            float x = fmass[r];
#pragma unroll
                            for (int d = 8; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                            if (lane == r) { wm[w * ROWS + r] = fref[r]; wl[w * ROWS + r] = x; }
                        }
                    } else {
#pragma unroll
                        for (int m = 0; m < RM; ++m)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                float x = mass[m][half];
                                x += __shfl_xor_sync(0xffffffffu, x, 1);
                                x += __shfl_xor_sync(0xffffffffu, x, 2);
                                if (r4 == 0) { wm[w * ROWS + m * 16 + half * 8 + g] = ref[m][half]; wl[w * ROWS + m * 16 + half * 8 + g] = x; }
                            }
                    }
                    if (lane == 0) stage_of[w] = had;
                }
                __syncthreads();
                const int w0 = first % NW, some = piece < NW ? piece : NW;       // warps w0, w0 + 1, ... (round the block)
                const bool whole = at.tile == 0 && piece == at.tiles;
                float* slot = p.part + (int64_t)(2 * blockIdx.x + (first_piece ? 0 : 1)) * ROWS * (p.V + 2);
                float joint = -INFINITY;                 // lane: of row `lane` (or lane & 15)
                const int jr = lane & (ROWS - 1);
#pragma unroll 4
                for (int i = 0, x = w0; i < some; ++i, x = x + 1 == NW ? 0 : x + 1) joint = fmaxf(joint, wm[x * ROWS + jr]);
                if (w == 0 && lane < ROWS) {
                    float sum = 0.f, f = 1.f;
#pragma unroll 1
                    for (int i = 0, x = w0; i < some; ++i, x = x + 1 == NW ? 0 : x + 1)
                        sum += joint == -INFINITY ? wl[x * ROWS + lane] : wl[x * ROWS + lane] * ex2_approx(wm[x * ROWS + lane] - joint);
                    int n, h;
                    if (row_of(p, at.unit, lane, n, h)) {
                        if (whole) {
                            const bool real = is_draft(p, at.b, n);
                            f = real ? finish_scale(sum) : -1.f;            // (a scale is never negative: -1 marks what is no draft)
                            if (p.lse) p.lse[((int64_t)at.b * p.N + n) * p.H + h] = real ? finish_lse(joint, sum) : -INFINITY;
                        } else {
                            *reinterpret_cast<float2*>(slot + ROWS * p.V + 2 * lane) = make_float2(joint, sum);
                        }
                    }
                    scale_of[lane] = f;
                }
                float f[RM][2];
                if constexpr (F32) {
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const float j = __shfl_sync(0xffffffffu, joint, r), y = j == -INFINITY ? 1.f : ex2_approx(fref[r] - j);
#pragma unroll
                        for (int i = 0; i < CW; ++i) fo[r][i] *= y;
                    }
                } else {
#pragma unroll
                    for (int m = 0; m < RM; ++m)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const float j = __shfl_sync(0xffffffffu, joint, m * 16 + half * 8 + g);
                            f[m][half] = j == -INFINITY ? 1.f : ex2_approx(ref[m][half] - j);
                        }
                }
#pragma unroll
                for (int c = 0; c < DV / S::cols; ++c) {
                    if (c > 0) __syncthreads();
                    if (had >= 0) {
                        float* own = reinterpret_cast<float*>(ring + had * S::stage);
                        if constexpr (F32) {
#pragma unroll
                            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                                for (int i = 0; i < CW; ++i) own[r * S::jrow + lane * CW + i] = fo[r][i];
                        } else
#pragma unroll
                        for (int m = 0; m < RM; ++m)
#pragma unroll
                            for (int d = 0; d < S::cols / 8; ++d)
#pragma unroll
                                for (int half = 0; half < 2; ++half)
                                    *reinterpret_cast<float2*>(own + (m * 16 + half * 8 + g) * S::jrow + d * 8 + 2 * r4) =
                                        make_float2(o[m][c * (S::cols / 8) + d][2 * half] * f[m][half], o[m][c * (S::cols / 8) + d][2 * half + 1] * f[m][half]);
                    }
                    __syncthreads();
#pragma unroll 1
                    for (int y = tid; y < ROWS * (S::cols / 4); y += NT) {
                        const int row = y / (S::cols / 4), q = y % (S::cols / 4) * 4, col = c * S::cols + q;
                        int n, h;
                        if (row_of(p, at.unit, row, n, h) && col < p.V) {
                            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                            for (int i = 0, x = w0; i < some; ++i, x = x + 1 == NW ? 0 : x + 1) {
                                const float4 v = *reinterpret_cast<const float4*>(sm + S::ring + (x * ST + stage_of[x]) * S::stage + (row * S::jrow + q) * 4);
                                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                            }
                            if (whole) {
                                const float z = scale_of[row];
                                T* to = reinterpret_cast<T*>(p.out) + (((int64_t)at.b * p.N + n) * p.H + h) * p.V + col;
                                if constexpr (F32) {
                                    *reinterpret_cast<float4*>(to) = z < 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(sum.x * z, sum.y * z, sum.z * z, sum.w * z);
                                } else {
                                    uint2 v = make_uint2(Frag<T>::pack(sum.x * z, sum.y * z), Frag<T>::pack(sum.z * z, sum.w * z));
                                    if (z < 0.f) v = make_uint2(0u, 0u);
                                    *reinterpret_cast<uint2*>(to) = v;
                                }
                            } else {
                                *reinterpret_cast<float4*>(slot + row * p.V + col) = sum;
                            }
                        }
                    }
                }
                if (tid == 0 && at.tile == 0) leave_task(p, at, x0 + first, x0, blockIdx.x, line, whole);
                first_piece = false;
                if (end == n_tiles) {
                    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
                    return;
                }
                const int b = at.b;
                at.tile += piece - 1;
                at.next(p);
                if (at.b != b) { bool d = false; draft_length(p, at.b, &d); bad |= d; }
                fetch_q(at);
                cp_async_commit();
                cp_async_wait<0>();
                __syncthreads();
                if (had >= 0 && (p.K < DK || p.V < DV)) {
                    for (int i = lane; i < S::stage / 16; i += 32) reinterpret_cast<uint4*>(ring + had * S::stage)[i] = make_uint4(0, 0, 0, 0);
                    __syncwarp();
                }
            } else {
                cp_async_wait<0>();                      // q, with the first tiles
                __syncthreads();
            }
            first = end;
            piece = min(n_tiles - first, at.tiles - at.tile);
            end = first + piece;
            had = -1;
            if constexpr (F32) {
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    fref[r] = -INFINITY;
                    fmass[r] = 0.f;
#pragma unroll
                    for (int i = 0; i < CW; ++i) fo[r][i] = 0.f;
                }
            } else {
#pragma unroll
            for (int m = 0; m < RM; ++m) {
                ref[m][0] = ref[m][1] = -INFINITY;
                mass[m][0] = mass[m][1] = 0.f;
#pragma unroll
                for (int d = 0; d < DV / 8; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[m][d][e] = 0.f;
                const uint32_t a = q_u + (m * 16 + (lane & 15)) * S::krow + (lane >> 4) * 16;
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks) ldmatrix4(qf[m][ks], a + ks * 32);
            }
            if (p.neg)
#pragma unroll
                for (int m = 0; m < RM; ++m)
#pragma unroll
                    for (int ks = 0; ks < DK / 16; ++ks)
#pragma unroll
                        for (int e = 0; e < 4; ++e) qf[m][ks][e] ^= 0x80008000u;
            }
        }

        // fetch tile k of this warp
        const int stage = k % ST;
        if (w + k * NW < n_tiles) {
            ahead.tile += step;
            step = NW;
            while (ahead.tile >= ahead.tiles) {
                ahead.tile -= ahead.tiles;
                if (++ahead.unit == p.Hkv * p.row_tiles) {
                    ahead.unit = 0;
                    ahead.enter(p, ahead.b + 1);
                }
                page_next = -2;
            }
            int page_of = k == 0 || page_next == -2 ? look(ahead) : page_next;
            const int kv = head_of(p, ahead.unit), pos0 = ahead.tile * kSlice;
            const uint32_t in0 = (uint32_t)pos0 - p.page.div((uint32_t)pos0) * p.page.d;
            uint32_t m = 0xffffu;
            const uint32_t kd = kdst + stage * S::stage, vd = vdst + stage * S::stage;
            __syncwarp();                  // every lane has read what the stage held
            if (ahead.tile < ahead.tiles - p.draft_tiles && pos0 + kSlice <= ahead.len && in0 + kSlice <= p.page.d && page_of >= 0 && page_of < p.pages) {
                // sixteen tokens of one page (the same one in every lane)
                const char* ks = p.ck + page_of * p.ck_page + (in0 + lane / KL) * p.ck_row + kv * p.ck_h + lane % KL * 16;
                const char* vs = p.cv + page_of * p.cv_page + (in0 + lane / VL) * p.cv_row + kv * p.cv_h + lane % VL * 16;
#pragma unroll
                for (int h = 0; h < KP; ++h) {
                    const char* src = ks + h * 512;
                    if (kcol(h))
#pragma unroll
                        for (int i = 0; i < kSlice * KL / 32; ++i, src += kstep) cp_async16(kd + i * (32 / KL) * S::krow + h * 512, src);
                }
#pragma unroll
                for (int h = 0; h < VP; ++h) {
                    const char* src = vs + h * 512;
                    if (vcol(h))
#pragma unroll
                        for (int i = 0; i < kSlice * VL / 32; ++i, src += vstep) cp_async16(vd + i * (32 / VL) * S::vrow + h * 512, src);
                }
            } else {
                const char *ks = p.q, *vs = p.q;         // (a row that is not there has no source)
                bool on = false;
                if (ahead.tile < ahead.tiles - p.draft_tiles) {
                    const int pos = pos0 + (lane & 15);
                    on = pos < ahead.len;
                    if (on && (page_of < 0 || page_of >= p.pages)) { bad = true; on = false; }
                    if (on) {
                        const int64_t in = (int64_t)(pos - p.page.div((uint32_t)pos) * p.page.d);
                        ks = p.ck + page_of * p.ck_page + in * p.ck_row + kv * p.ck_h;
                        vs = p.cv + page_of * p.cv_page + in * p.cv_row + kv * p.cv_h;
                    }
                } else {
                    const int n = (ahead.tile - (ahead.tiles - p.draft_tiles)) * kSlice + (lane & 15);
                    on = n < p.N && is_draft(p, ahead.b, n);
                    if (on) {
                        ks = p.k + ahead.b * p.k_b + n * p.k_n + kv * p.k_h;
                        vs = p.v + ahead.b * p.v_b + n * p.v_n + kv * p.v_h;
                    }
                }
                m = __ballot_sync(0xffffffffu, on) & 0xffffu;
#pragma unroll 1
                for (int i = 0; i < kSlice * KL / 32; ++i) {
                    const int j = i * (32 / KL) + lane / KL;
                    const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(ks), j));
#pragma unroll
                    for (int h = 0; h < KP; ++h)
                        if (kcol(h)) cp_async16_or_zero(kd + i * (32 / KL) * S::krow + h * 512, (m >> j & 1) ? src + lane % KL * 16 + h * 512 : p.q, m >> j & 1);
                }
#pragma unroll 1
                for (int i = 0; i < kSlice * VL / 32; ++i) {
                    const int j = i * (32 / VL) + lane / VL;
                    const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vs), j));
#pragma unroll
                    for (int h = 0; h < VP; ++h)
                        if (vcol(h)) cp_async16_or_zero(vd + i * (32 / VL) * S::vrow + h * 512, (m >> j & 1) ? src + lane % VL * 16 + h * 512 : p.q, m >> j & 1);
                }
            }
            keys_of = (keys_of & ~(0xffffull << (16 * stage))) | (uint64_t)m << (16 * stage);
            Place pl = ahead;
            pl.tile += NW;
            page_next = look(pl);          // (of no use where the unit ends before: looked up again)
        }
        cp_async_commit();
        if (t < 0) continue;

        const int cached = at.tiles - p.draft_tiles, tile = at.tile + (mine - first), cur = t % ST;
        const bool draft = tile >= cached;
        had = cur;
        cp_async_wait<ST - 1>();
        __syncwarp();
        const uint32_t kbase = ring_u + cur * S::stage, vbase = kbase + kSlice * S::krow;
        const uint32_t keys = (uint32_t)(keys_of >> (16 * cur)) & 0xffffu;
        if constexpr (F32) {
            // Lane x has key x & 15, and of every row half the elements.
            const int key = lane & 15;
            float s[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) s[r] = 0.f;
            const float* kk = reinterpret_cast<const float*>(sm + (kbase - smem_u32(sm)) + key * S::krow) + (lane >> 4) * (DK / 2);
            const float* qq = reinterpret_cast<const float*>(sm + S::q) + (lane >> 4) * (DK / 2);
#pragma unroll 4
            for (int d = 0; d < DK / 2; d += 4) {
                const float4 x = *reinterpret_cast<const float4*>(kk + d);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const float4 y = *reinterpret_cast<const float4*>(qq + r * (S::krow / 4) + d);
                    s[r] = fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, s[r]))));
                }
            }
            uint32_t own = keys;                          // which keys row `lane` reads
            if (draft) {
                int n, h;
                own = lane < ROWS && row_of(p, at.unit, lane, n, h) ? keys & (uint32_t)draft_mask(p, at.b, n, (tile - cached) * kSlice, &bad) : 0u;
            }
            bool above = false;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                s[r] += __shfl_xor_sync(0xffffffffu, s[r], 16);
                const uint32_t seen = draft ? __shfl_sync(0xffffffffu, own, r) : keys;
                s[r] = (seen >> key & 1) ? s[r] * p.c : -INFINITY;
                above |= s[r] > fref[r] + kLag<T>;
            }
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    float x = s[r];
#pragma unroll
                    for (int d = 8; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    const float now = fmaxf(fref[r], x), keep = now == -INFINITY ? 1.f : ex2_approx(fref[r] - now);
                    fref[r] = now;
                    fmass[r] *= keep;
#pragma unroll
                    for (int i = 0; i < CW; ++i) fo[r][i] *= keep;
                }
            }
            float* pw = reinterpret_cast<float*>(sm + S::p) + w * ROWS * kSlice;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float e = ex2_approx(s[r] - (fref[r] == -INFINITY ? 0.f : fref[r]));
                fmass[r] += e;
                if (lane < 16) pw[r * kSlice + lane] = e;
            }
            __syncwarp();
            const float* vv = reinterpret_cast<const float*>(sm + (vbase - smem_u32(sm))) + lane * CW;
#pragma unroll
            for (int j = 0; j < kSlice; j += 4) {
                float x[4][CW];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (CW >= 4) {
#pragma unroll
                        for (int c = 0; c < CW; c += 4) *reinterpret_cast<float4*>(x[i] + c) = *reinterpret_cast<const float4*>(vv + (j + i) * (S::vrow / 4) + c);
                    } else *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(vv + (j + i) * (S::vrow / 4));
                }
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const float4 y = *reinterpret_cast<const float4*>(pw + r * kSlice + j);
                    const float ys[4] = {y.x, y.y, y.z, y.w};
                    const uint32_t seen = draft ? __shfl_sync(0xffffffffu, own, r) >> j : 0xfu;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!(seen >> i & 1)) continue;       // a draft's values, whatever they are, stay with those that read it
#pragma unroll
                        for (int c = 0; c < CW; ++c) fo[r][c] = fmaf(ys[i], x[i][c], fo[r][c]);
                    }
                }
            }
            __syncwarp();
        } else {
        uint32_t spoilt = 0;
        if (draft) {
#pragma unroll 1
            for (int x = lane; x < kSlice * (DV / 8); x += 32)
                if (take_out<T>(vbase + x / (DV / 8) * S::vrow + x % (DV / 8) * 16)) spoilt |= 1u << (x / (DV / 8));
            spoilt = __reduce_or_sync(0xffffffffu, spoilt);
            __syncwarp();
        }
        float s[RM][2][4];
#pragma unroll
        for (int m = 0; m < RM; ++m)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[m][nt][e] = 0.f;
        {
            const uint32_t a = kbase + (((lane >> 4) << 3) + (lane & 7)) * S::krow + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
                uint32_t b[4];
                ldmatrix4(b, a + ks * 32);
#pragma unroll
                for (int m = 0; m < RM; ++m) {
                    Frag<T>::mma(s[m][0], qf[m][ks][0], qf[m][ks][1], qf[m][ks][2], qf[m][ks][3], b[0], b[1]);
                    Frag<T>::mma(s[m][1], qf[m][ks][0], qf[m][ks][1], qf[m][ks][2], qf[m][ks][3], b[2], b[3]);
                }
            }
        }
        uint32_t seen[RM][2];
#pragma unroll
        for (int m = 0; m < RM; ++m) seen[m][0] = seen[m][1] = keys;
        if (draft) {
#pragma unroll 1
            for (int m = 0; m < RM; ++m) {
                int n, h;
                uint32_t own = 0;
                if (lane < 16 && row_of(p, at.unit, m * 16 + lane, n, h)) own = (uint32_t)draft_mask(p, at.b, n, (tile - cached) * kSlice, &bad) & 0xffffu;
                const uint32_t lo = __shfl_sync(0xffffffffu, own, g), hi = __shfl_sync(0xffffffffu, own, g + 8);
#pragma unroll
                for (int i = 0; i < RM; ++i) if (i == m) { seen[i][0] &= lo; seen[i][1] &= hi; }
            }
        }
        if (draft || keys != 0xffffu) {
#pragma unroll
            for (int m = 0; m < RM; ++m)
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(seen[m][e >> 1] >> (nt * 8 + 2 * r4 + (e & 1)) & 1)) s[m][nt][e] = -INFINITY;
        }
        uint32_t pf[RM][4];
#pragma unroll
        for (int m = 0; m < RM; ++m) {
            float top[2];
#pragma unroll
            for (int half = 0; half < 2; ++half)
                top[half] = p.c * fmaxf(fmaxf(s[m][0][2 * half], s[m][0][2 * half + 1]), fmaxf(s[m][1][2 * half], s[m][1][2 * half + 1]));
            if (__any_sync(0xffffffffu, top[0] > ref[m][0] + (kLag<T> + kBias<T>) || top[1] > ref[m][1] + (kLag<T> + kBias<T>))) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float x = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    const float now = fmaxf(ref[m][half], x - kBias<T>);
                    const float keep = now == -INFINITY ? 1.f : ex2_approx(ref[m][half] - now);
                    ref[m][half] = now;
                    mass[m][half] *= keep;
#pragma unroll
                    for (int d = 0; d < DV / 8; ++d) {
                        o[m][d][2 * half] *= keep;
                        o[m][d][2 * half + 1] *= keep;
                    }
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float base = ref[m][half] == -INFINITY ? 0.f : -ref[m][half];
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = ex2_approx(fmaf(s[m][i >> 1][2 * half + (i & 1)], p.c, base));
                mass[m][half] += (e[0] + e[1]) + (e[2] + e[3]);
                pf[m][half] = Frag<T>::pack(e[0], e[1]);
                pf[m][half + 2] = Frag<T>::pack(e[2], e[3]);
            }
        }
        {
            const uint32_t a = vbase + ((((lane >> 3) & 1) << 3) + (lane & 7)) * S::vrow + (lane >> 4) * 16;
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
                uint32_t b[4];
                ldmatrix4_trans(b, a + d * 32);
#pragma unroll
                for (int m = 0; m < RM; ++m) {
                    Frag<T>::mma(o[m][2 * d], pf[m][0], pf[m][1], pf[m][2], pf[m][3], b[0], b[1]);
                    Frag<T>::mma(o[m][2 * d + 1], pf[m][0], pf[m][1], pf[m][2], pf[m][3], b[2], b[3]);
                }
            }
        }
        if (spoilt)
#pragma unroll 1
            for (int j = 0; j < kSlice; ++j) {
                if (!(spoilt >> j & 1)) continue;
                const char* v = p.v + at.b * p.v_b + ((tile - cached) * kSlice + j) * p.v_n + head_of(p, at.unit) * p.v_h;
#pragma unroll
                for (int m = 0; m < RM; ++m)
#pragma unroll
                    for (int d = 0; d < DV / 8; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int col = d * 8 + 2 * r4 + (e & 1);
                            if ((seen[m][e >> 1] >> j & 1) && col < p.V) o[m][d][e] = put_back<T>(o[m][d][e], v, col);
                        }
            }
        }
    }
}

// ---- fp32, more than 16 query rows: FFMA -------------------------------------------------------------------------------------

// 64 query rows a block against tiles of 64 keys, four warps of 16 rows each.  A thread has 8 rows and, of the scores, the keys
// kg, kg + 16, .. of the tile, of the sums the columns 4 cg .. 4 cg + 3 of every 64 (kg = cg = lane & 15): per 64 products it reads 4 to 6
// times 16 bytes of shared memory, so that the FMA pipes bound it and not the reads.  A warp's weights stay in it.  The keys of the next tile come
// by cp.async while the values are multiplied, the values while the scores are; pieces of 16 bytes are swizzled so that the lanes of a
// read meet in no bank.  Measured, 4 requests of 16384, 4 heads of 128, 256 rows: 935 us, 37 TFLOP/s (slices of sixteen rows: 1983 us);
// seven in ten issue slots are taken, seven in ten of those by products.  Products of two at a time in packed instructions change it by 2%.
constexpr int kFmaRows = 64, kFmaThreads = 128;
template <int D> struct FmaShape {
    static constexpr int q = 0, k = q + kFmaRows * D * 4, v = k + kTile * D * 4, p = v + kTile * D * 4, mask = p + kFmaRows * kTile * 4,
                         there = mask + kFmaRows * 8, total = there + 16;
};

template <int D>
__global__ void __launch_bounds__(kFmaThreads, D > 128 ? 1 : 2) draft_fma_kernel(const __grid_constant__ DraftParams p) {
    using S = FmaShape<D>;
    constexpr int CJ = D / 64;                          // float4s of a thread's columns
    extern __shared__ __align__(128) unsigned char sm[];
    uint64_t* mask = reinterpret_cast<uint64_t*>(sm + S::mask);              // which drafts of the tile a row reads
    uint16_t* there = reinterpret_cast<uint16_t*>(sm + S::there);            // [2][4]: which keys the tile has, this tile's and the next one's
    const uint32_t base = smem_u32(sm);
    chain_enter();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rg = lane >> 4, kg = lane & 15;
    Place at;
    Line line;
    int64_t x0, x1;
    if (tid == 0 && !p.by_unit && !p.whole) p.tasks[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (!find_part<kFmaThreads>(p, at, line, x0, x1)) return;
    bool bad = false;
    { bool b = false; draft_length(p, at.b, &b); bad |= b; }
    // Where the keys and values of a tile are: lane j (and j + 16) knows key 16 w + j.
    const char *kp = nullptr, *vp = nullptr;
    uint32_t has = 0;
    auto look = [&](const Place& pl, int buf) {
        kp = vp = p.q;
        has = __ballot_sync(0xffffffffu, key_row(p, pl, head_of(p, pl.unit), w * 16 + kg, kp, vp, &bad)) & 0xffffu;
        if (lane == 0) there[buf * 4 + w] = (uint16_t)has;
    };
    // ... and this warp's sixteen of them, to shared memory
    auto copy = [&](const char* rows, uint32_t dst, int width, bool swizzled) {
#pragma unroll 4
        for (int j = 0; j < 16; ++j) {
            const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(rows), j));
            const bool on = has >> j & 1;
            for (int c = lane; c * 4 < width; c += 32)
                cp_async16_or_zero(dst + (w * 16 + j) * (D * 4) + (swizzled ? c ^ (j & 7) : c) * 16, on ? src + c * 16 : p.q, on);
        }
        cp_async_commit();
    };
    look(at, 0);
    copy(kp, base + S::k, p.K, true);
    float m[8], mass[8], o[8][CJ * 4];
    int first_tile = at.tile;                           // of the unit's part in this block
    bool fresh = true, first_piece = true;
    int buf = 0;
    const float* sq = reinterpret_cast<const float*>(sm + S::q) + (w * 16 + rg * 8) * D;
    const float* sk = reinterpret_cast<const float*>(sm + S::k) + kg * D;
    const float* sv = reinterpret_cast<const float*>(sm + S::v) + kg * 4;
    float* sp = reinterpret_cast<float*>(sm + S::p) + w * (16 * kTile) + rg * 8;              // [key][16 rows]
    for (int64_t x = x0; x < x1; ++x, buf ^= 1) {
        if (fresh) {
            fresh = false;
            first_tile = at.tile;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                m[r] = -INFINITY;
                mass[r] = 0.f;
#pragma unroll
                for (int i = 0; i < CJ * 4; ++i) o[r][i] = 0.f;
            }
#pragma unroll 1
            for (int j = 0; j < 16; ++j) {
                int n, h;
                const bool on = row_of(p, at.unit, w * 16 + j, n, h);
                for (int c = lane; c * 4 < p.K; c += 32)
                    cp_async16_or_zero(base + S::q + (w * 16 + j) * (D * 4) + (c ^ (j >> 3)) * 16, on ? p.q + at.b * p.q_b + n * p.q_n + h * p.q_h + c * 16 : p.q, on);
            }
            cp_async_commit();
        }
        copy(vp, base + S::v, p.V, false);
        const int cached = at.tiles - p.draft_tiles, tile0 = (at.tile - cached) * kTile;
        const bool draft = tile0 >= 0;
        bool idle = false;                              // a chain's drafts behind the rows of this tile
        if (draft) {
            int n, h;
            if (tid < kFmaRows) mask[tid] = row_of(p, at.unit, tid, n, h) ? draft_mask(p, at.b, n, tile0, &bad) : 0ull;
            (void)row_of(p, at.unit, kFmaRows - 1, n, h);
            idle = !p.parents && tile0 > n;
        }
        cp_async_wait<1>();                             // the keys, and q
        __syncthreads();
        if (!idle) {
            float s[8][4];
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[r][j] = 0.f;
#pragma unroll 2
            for (int c = 0; c < p.K / 4; ++c) {
                float4 a[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = *reinterpret_cast<const float4*>(sk + j * 16 * D + (c ^ (kg & 7)) * 4);
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float4 y = *reinterpret_cast<const float4*>(sq + r * D + (c ^ rg) * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[r][j] = fmaf(y.w, a[j].w, fmaf(y.z, a[j].z, fmaf(y.y, a[j].y, fmaf(y.x, a[j].x, s[r][j]))));
                }
            }
            const uint64_t keys = *reinterpret_cast<const uint64_t*>(there + buf * 4);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const uint64_t seen = (draft ? keys & mask[w * 16 + rg * 8 + r] : keys) >> kg;
                float top = m[r];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[r][j] = (seen >> (16 * j) & 1) ? s[r][j] * p.c : -INFINITY;
                    top = fmaxf(top, s[r][j]);
                }
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float ref = top == -INFINITY ? 0.f : top, keep = ex2_approx(m[r] - ref);
                m[r] = top;
#pragma unroll
                for (int j = 0; j < 4; ++j) s[r][j] = ex2_approx(s[r][j] - ref);
                mass[r] = fmaf(mass[r], keep, (s[r][0] + s[r][1]) + (s[r][2] + s[r][3]));
                if (keep != 1.f)
#pragma unroll
                    for (int i = 0; i < CJ * 4; ++i) o[r][i] *= keep;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 8; r += 4) *reinterpret_cast<float4*>(sp + (kg + 16 * j) * 16 + r) = make_float4(s[r][j], s[r + 1][j], s[r + 2][j], s[r + 3][j]);
        }
        __syncthreads();                                // all have read the keys
        Place next = at;
        if (x + 1 < x1) {
            next.next(p);
            if (next.b != at.b) { bool d = false; draft_length(p, next.b, &d); bad |= d; }
            look(next, buf ^ 1);
            copy(kp, base + S::k, p.K, true);
        } else {
            cp_async_commit();
        }
        cp_async_wait<1>();                             // the values
        __syncthreads();
        if (!idle) {
            auto add = [&](auto some) {
#pragma unroll 4
                for (int key = 0; key < kTile; ++key) {
                    float y[8];
                    *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(sp + key * 16);
                    *reinterpret_cast<float4*>(y + 4) = *reinterpret_cast<const float4*>(sp + key * 16 + 4);
#pragma unroll
                    for (int i = 0; i < CJ; ++i) {
                        const float4 a = *reinterpret_cast<const float4*>(sv + key * D + i * 64);
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            // (a draft's values, whatever they are, stay with those that read it)
                            if (decltype(some)::value && !(mask[w * 16 + rg * 8 + r] >> key & 1)) continue;
                            o[r][4 * i] = fmaf(y[r], a.x, o[r][4 * i]);
                            o[r][4 * i + 1] = fmaf(y[r], a.y, o[r][4 * i + 1]);
                            o[r][4 * i + 2] = fmaf(y[r], a.z, o[r][4 * i + 2]);
                            o[r][4 * i + 3] = fmaf(y[r], a.w, o[r][4 * i + 3]);
                        }
                    }
                }
            };
            if (draft) add(std::true_type{}); else add(std::false_type{});
        }
        const bool done = at.tile + 1 == at.tiles;
        if (done || x + 1 == x1) {                      // the unit ends, or this block's part of it
            const bool whole = done && first_tile == 0;
            float* slot = p.part + (int64_t)(2 * blockIdx.x + (first_piece ? 0 : 1)) * kFmaRows * (p.V + 2);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float sum = mass[r];
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const int row = w * 16 + rg * 8 + r;
                int n, h;
                if (!row_of(p, at.unit, row, n, h)) continue;
                const bool real = is_draft(p, at.b, n);
                const float inv = whole ? (real ? finish_scale(sum) : 0.f) : 1.f;
                const int64_t at_out = ((int64_t)at.b * p.N + n) * p.H + h;
                float* to = whole ? reinterpret_cast<float*>(p.out) + at_out * p.V : slot + row * p.V;
#pragma unroll
                for (int i = 0; i < CJ; ++i) {
                    const int col = i * 64 + kg * 4;
                    if (col >= p.V) continue;
                    float4 y = make_float4(o[r][4 * i] * inv, o[r][4 * i + 1] * inv, o[r][4 * i + 2] * inv, o[r][4 * i + 3] * inv);
                    if (whole && !real) y = make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4*>(to + col) = y;
                }
                if (kg == 0) {
                    if (!whole) *reinterpret_cast<float2*>(slot + kFmaRows * p.V + 2 * row) = make_float2(m[r], sum);
                    else if (p.lse) p.lse[at_out] = real ? finish_lse(m[r], sum) : -INFINITY;
                }
            }
            if (tid == 0 && first_tile == 0) leave_task(p, at, x - at.tile, x0, blockIdx.x, line, whole);
            first_piece = false;
            fresh = true;
        }
        at = next;
        __syncthreads();                                // the values and masks have been read
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
}

// ---- 16-bit types, more than 32 query rows (16 where rows are wider than 64): tcgen05 -----------------------------------------------------------------------------------

// 128 or 256 query rows a block against tiles of 128 keys, which come from HBM once for all of them.  Per job (a tile and 128 rows, the lanes
// of tensor memory): S = Q K^T (operands in shared memory, accumulator in tensor memory), P = 2^(cS - reference) by a thread a row, written
// over S in 16 bits, O += P V with P read from tensor memory.  Two halves with an S and an O of their own take turns, so that one's softmax
// runs beside the other's products: with more than 128 rows each has 128 of them and all tiles, with fewer both have the same rows and
// every other tile, and are joined at the end.  Tensor memory: S and O of each half, 128 columns each; shared memory: Q (64 KB), three
// stages of K and two of V (32 KB).  Roles: warps 0-3 and 4-7 the softmax of a half, 8 the products, 9-11 the copies.
// At 256 rows of 128 a tile is 16.8 MFLOP, 2048 cycles of the tensor pipe, and 32768 exponentials, 2048 cycles of the special function
// units: the two bound it alike, HBM (64 KB a tile) does below about 250 rows.  A tile of 256 rows takes 3100 cycles as it is, a part
// 37000 more (cold, under a profiler); no unit's counter is above half.  Measured in bf16, 128 wide: 4 requests of 16384, 8 heads, chunks of
// 512 drafts with 4 query heads each: 635 us, 880 TFLOP/s; 8 of 65536, 4 heads, 256 rows: 303 to 313 us, 880 to 907 TFLOP/s, 128 rows 215 us, 5.0 TB/s.
// A row's weights in a tile may sum to kTcMost before the reference follows (a maximum per tile costs a fifth of the softmax; the sum is there
// anyway); a reference is set kTcBias below a tile's maximum, the first one, where all keys of the tile are read, below that of its first sixteen scores:
// later ones may be any distance above it, and the sum and exp2_poly's largest exponent tell.  bf16 has fp32's range; fp16 ends at 65504 and keeps all its digits down to 2^-14.
template <typename T> constexpr float kTcMost = 65536.f;
template <> constexpr float kTcMost<__half> = 60000.f;
template <typename T> constexpr float kTcBias = 0.f;
template <> constexpr float kTcBias<__half> = 6.f;
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 ra, rb, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nadd.rn.f32x2 rd, ra, rb;\nmov.b64 {%0, %1}, rd;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
constexpr int kTcTile = 128, kTcThreads = 384, kTcProducers = 3, kTcMma = 8, kTcCopy = 9;        // (warps)
constexpr int kTcWaitCap = 1 << 20, kTcPolyEvery = 4;

__device__ __forceinline__ uint32_t tc_idesc(bool bf16, bool negate, bool v_major, int n) {
    // fp32 accumulator; A and B f16 (0) or bf16 (1); A negated; B with N (1) or K (0) contiguous; N / 8; M = 128
    const uint32_t type = bf16 ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | (negate ? 1u : 0u) << 13 | (v_major ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
// Descriptors of operands in shared memory: rows of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes; `lead` is the distance of 64-element
// blocks along a contiguous N.  The address is in the low word, so that a step along the operand is one addition.
__device__ __forceinline__ uint32_t tc_desc(uint32_t addr, uint32_t lead) { return addr >> 4 | (lead >> 4) << 16; }
constexpr uint32_t kTcDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %4, 0;\nmov.b64 da, {%1, %5};\nmov.b64 db, {%2, %5};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(kTcDescHigh) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 db;\nsetp.ne.b32 p, 1, 0;\nmov.b64 db, {%2, %4};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(kTcDescHigh) : "memory");
}
// One lane of the warp, always the same (and the compiler knows that it is one: the operands of its products are uniform).
__device__ __forceinline__ bool elect_one() {
    uint32_t x;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(x));
    return x != 0;
}
// 2^t on the FMA pipes, two at a time: t = n + f with n the nearest integer (it appears in the low bits of t + 1.5 * 2^23), 2^f by a polynomial
// of degree 5 (fitted to the smallest largest relative error over [-1/2, 1/2], 2.3e-7 in fp32), n added to the exponent.  What is below -126
// comes out as 2^-126.  Above 126, where n runs through the exponent into the sign, the result means nothing and may be small: `most` is the
// largest t (NaN if one is), by which the caller has to tell.  (Telling costs 2% of tree_16k, 145 -> 149 us, and 1% of chunk_8k; cutting t off
// above as well 3.5% of both.)
constexpr float kPolyMost = 126.f;
__device__ __forceinline__ float2 exp2_poly(float2 t, float& most) {
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(t.x));
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(t.y));
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(t.x), "f"(t.y));
    const float2 big = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);
    const float2 r = fadd2(t, big), n = fadd2(r, minus), f = ffma2(n, make_float2(-1.f, -1.f), t);
    float2 y = ffma2(make_float2(0.0013276470126584172f, 0.0013276470126584172f), f, make_float2(0.009675540961325169f, 0.009675540961325169f));
    y = ffma2(y, f, make_float2(0.05550713092088699f, 0.05550713092088699f));
    y = ffma2(y, f, make_float2(0.24022120237350464f, 0.24022120237350464f));
    y = ffma2(y, f, make_float2(0.6931469440460205f, 0.6931469440460205f));
    y = ffma2(y, f, make_float2(1.0000001192092896f, 1.0000001192092896f));
    return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(r.x) << 23)), __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(r.y) << 23)));
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
#define TC_R8(x, i) "=r"((x)[i]), "=r"((x)[i + 1]), "=r"((x)[i + 2]), "=r"((x)[i + 3]), "=r"((x)[i + 4]), "=r"((x)[i + 5]), "=r"((x)[i + 6]), "=r"((x)[i + 7])
#define TC_U8(x, i) "+r"((x)[i]), "+r"((x)[i + 1]), "+r"((x)[i + 2]), "+r"((x)[i + 3]), "+r"((x)[i + 4]), "+r"((x)[i + 5]), "+r"((x)[i + 6]), "+r"((x)[i + 7])
#define TC_W8(x, i) "r"((x)[i]), "r"((x)[i + 1]), "r"((x)[i + 2]), "r"((x)[i + 3]), "r"((x)[i + 4]), "r"((x)[i + 5]), "r"((x)[i + 6]), "r"((x)[i + 7])
// 16 columns of this warp's 32 lanes, a lane a thread; not to be read before tc_wait_ld
__device__ __forceinline__ void tc_ld16(uint32_t (&x)[16], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : TC_R8(x, 0), TC_R8(x, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_wait_ld(uint32_t (&x)[16]) { asm volatile("tcgen05.wait::ld.sync.aligned;\n" : TC_U8(x, 0), TC_U8(x, 8)::"memory"); }
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr), TC_W8(x, 0), TC_W8(x, 8) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
                 "%29,%30,%31,%32};\n" ::"r"(addr), TC_W8(x, 0), TC_W8(x, 8), TC_W8(x, 16), TC_W8(x, 24) : "memory");
}

// The caches as [page][head][token][element] and the drafts' k, v as [request][head][draft][element], boxes of 16 tokens and 128 bytes; q as
// [request][draft][head][element], boxes of a group's heads of 128 / G drafts.
struct TcMaps { CUtensorMap k, v, kb, vb, dk, dv, q; };      // kb, vb: boxes of box_rows tokens

template <int DK, int DV> struct TcShape {
    static constexpr int kst = kTcTile * DK * 2, vst = kTcTile * DV * 2, qhalf = 128 * DK * 2;
    static constexpr int vstages = DK + DV > 192 ? 2 : 3, kstages = 3;
    static constexpr int q = 0, k = 2 * qhalf, v = k + kstages * kst, end = v + vstages * vst;
    static constexpr int bars = end, valid = bars + 256, spoilt = valid + 8 * 16, slot = spoilt + 8 * 16, swap = slot + 16, total = swap + 128 * 8 + 1024;
    static_assert(total + 128 <= 232448, "");
};
// mbarriers
enum { kQFull = 0, kQEmpty, kSFull, kPReady = kSFull + 2, kOFull = kPReady + 2, kKFull = kOFull + 2, kKEmpty = kKFull + 3, kVFull = kKEmpty + 3, kVEmpty = kVFull + 3, kRaw = kVEmpty + 3, kDone = kRaw + kTcProducers, kTcBars };
static_assert(kTcBars * 8 <= 256, "");

template <typename T, int DK, int DV>
__global__ void __launch_bounds__(kTcThreads, 1) draft_tc_kernel(const __grid_constant__ DraftParams p, const __grid_constant__ TcMaps maps) {
    using S = TcShape<DK, DV>;
    constexpr int KS = S::kstages, VS = S::vstages;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char sm_raw[];
    unsigned char* sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::bars);
    uint32_t* valid = reinterpret_cast<uint32_t*>(sm + S::valid);            // [8][4]: which keys a tile has
    uint32_t* spoilt = reinterpret_cast<uint32_t*>(sm + S::spoilt);          // [8][4]: drafts with values that are not finite
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + S::slot);
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    if (tid == 0) {
        mbar_init(bars + kQFull, kTcProducers); mbar_init(bars + kQEmpty, 1);
        for (int i = 0; i < 2; ++i) { mbar_init(bars + kSFull + i, 1); mbar_init(bars + kPReady + i, 128); mbar_init(bars + kOFull + i, 1); }
        for (int i = 0; i < 3; ++i) {
            mbar_init(bars + kKFull + i, 1); mbar_init(bars + kKEmpty + i, 1);
            mbar_init(bars + kVFull + i, 1); mbar_init(bars + kVEmpty + i, 1);
        }
        for (int i = 0; i < kTcProducers; ++i) mbar_init(bars + kRaw + i, 1);
        mbar_init(bars + kDone, 1);
        fence_barrier_init();
    }
    if (tid < 32) spoilt[tid] = 0;
    chain_enter();
    Place at;
    Line line;
    int64_t x0, x1;
    if (tid == 0 && !p.by_unit && !p.whole) p.tasks[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (!find_part<kTcThreads>(p, at, line, x0, x1)) return;
    const int n_tiles = (int)(x1 - x0);
    if (w == kTcMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;                     // columns: S of half 0, S of half 1, O of half 0, O of half 1
    bool bad = false, late = false;
    auto wait = [&](int bar, uint32_t parity) {
        if (!late && !mbar_wait_bounded(bars + bar, parity, kTcWaitCap)) late = true;      // (then nothing is waited for any more: wrong numbers, reported, no hang)
    };
    // Tiles that have work: of a chain's drafts not those behind the row tile's last (they stand in the line all the same).
    auto useful = [&](const Place& pl, int tiles) {
        if (p.parents) return tiles;
        const int rt = pl.unit - head_of(p, pl.unit) * p.row_tiles, last = min((int)p.group.div((uint32_t)(rt * p.rows + p.rows - 1)), p.N - 1);
        return max(0, min(tiles, pl.tiles - p.draft_tiles + last / kTcTile + 1 - pl.tile));
    };
    auto two_halves = [&](const Place& pl) { return p.N * p.G - (pl.unit - head_of(p, pl.unit) * p.row_tiles) * p.rows > 128 && p.rows > 128; };

    if (w >= kTcCopy) {
        // ---- copies.  (No warp may come to a stage's next tile but one before the next is done with: it would take the phase before for its own.)
        constexpr int KL = DK / 8, VL = DV / 8;
        const uint32_t base = smem_u32(sm);
        const int cw = w - kTcCopy;
        int g = 0, unit_no = 0, done = 0;
        uint32_t raws = 0;
        int last = -1;
        // where lane's piece of row r goes within a 128-row operand: 64 columns to a block of 128-byte rows, 16-byte pieces swizzled by the row
        auto place_of = [&](int r, int c) { return (uint32_t)((c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); };
        auto tell = [&](int bar, uint32_t bytes) { if (lane == 0) mbar_arrive_expect_tx(bars + bar, bytes); };
        // `blocks` boxes of 64 columns; by one lane
        auto box = [&](const CUtensorMap& map, int blocks, int bar, uint32_t dst, int row, int head, int page) {
            for (int blk = 0; blk < blocks; ++blk)
                asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(
                                 dst + blk * (128 * 128)), "l"(&map), "r"(blk * 64), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bars + bar)) : "memory");
        };
        // (rows of values that are not there become zero; rows of keys may hold anything, their scores are masked)
        auto copy_rows = [&](auto lanes_, uint32_t dst, const unsigned long long (&rows)[4], const uint32_t (&words)[4], uint32_t boxes, int width, bool all_rows) {
            constexpr int lanes = decltype(lanes_)::value, per = 32 / lanes;             // lanes of a row, rows at a time
            const int c = lane % lanes, mine = lane / lanes;
            const bool col = c * 8 < width;
            const uint32_t to = dst + (c >> 3) * (128 * 128) + mine * 128, piece = (uint32_t)((c & 7) ^ mine);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if ((boxes >> (2 * q) & 3u) == 3u) continue;
#pragma unroll
                for (int r = 0; r < 32; r += per) {
                    if (boxes >> (2 * q + (r >> 4)) & 1u) continue;
                    const unsigned long long src = __shfl_sync(0xffffffffu, rows[q], r + mine);
                    const bool on = (words[q] >> (r + mine) & 1u) && col;
                    if (!all_rows && !(words[q] >> r & ((1u << per) - 1u))) continue;
                    cp_async16_or_zero(to + (q * 32 + r) * 128 + ((piece ^ (r & 7)) << 4), on ? reinterpret_cast<const char*>(src) + c * 16 : p.q, on);
                }
            }
        };
        while (done < n_tiles) {
            const int share = min(n_tiles - done, at.tiles - at.tile), piece = useful(at, share), cached = at.tiles - p.draft_tiles, kv = head_of(p, at.unit);
            if (cw == 0) { bool b = false; draft_length(p, at.b, &b); bad |= b; }
            if (piece == 0) {
                done += share;
                at.tile += share - 1;
                at.next(p);
                continue;
            }
            const int row0 = (at.unit - kv * p.row_tiles) * p.rows, halves = two_halves(at) ? 2 : 1;
            wait(kQEmpty, (unit_no & 1) ^ 1);
            if (p.boxes & 2) {                            // whole drafts to a half: a box of the heads of 128 / G drafts
                if (cw == 0) {
                    tell(kQFull, halves * S::qhalf);
                    __syncwarp();
                    if (elect_one()) for (int i = 0; i < halves; ++i)
                        box(maps.q, DK / 64, kQFull, base + S::q + i * S::qhalf, kv * p.G, (int)p.group.div((uint32_t)(row0 + i * 128)), at.b);
                } else {
                    tell(kQFull, 0);
                }
            } else {
#pragma unroll 2
                for (int r0 = cw * (32 / KL); r0 < halves * 128; r0 += kTcProducers * (32 / KL)) {
                    const int r = r0 + lane / KL, c = lane % KL;
                    int n, h;
                    const bool on = row_of(p, at.unit, r, n, h) && c * 8 < p.K;
                    if (r < halves * 128)
                        cp_async16_or_zero(base + S::q + (r >> 7) * S::qhalf + place_of(r & 127, c), on ? p.q + at.b * p.q_b + n * p.q_n + h * p.q_h + c * 16 : p.q, on);
                }
                cp_async_commit();
                cp_async_wait<0>();
                fence_proxy_async();
                __syncwarp();
                tell(kQFull, 0);
            }
            // warp 0 the keys, in order; warps 1 and 2 the values of even and odd tiles
            const bool values = cw > 0;
            int j = values ? (cw - 1 + g) & 1 : 0;
            const int jstep = values ? 2 : 1, lanes = values ? VL : KL, width = values ? p.V : p.K;
            int late_bar = -1;
            uint32_t late_bytes = 0;
            int looked = -1, page = -1;                   // lane i < 8: the page of slice i of the next tile
            auto look = [&](int tile) {
                const int pos = tile * kTcTile + (lane & 7) * 16;
                looked = tile;
                page = tile < cached && pos < at.len ? __ldg(p.table + (int64_t)at.b * p.table_stride + p.page.div((uint32_t)pos)) : -1;
            };
            for (; j < piece; j += jstep) {
                const int t = g + j, tile = at.tile + j, st = values ? t % VS : t % KS, turn = values ? t / VS : t / KS;
                const int full = (values ? kVFull : kKFull) + st, empty = (values ? kVEmpty : kKEmpty) + st;
                const uint32_t dst = base + (values ? S::v + st * S::vst : S::k + st * S::kst);
                const bool draft = tile >= cached;
                const int n0 = (tile - cached) * kTcTile;
                if (looked != tile) look(tile);
                // Slices of sixteen keys that are one box of a tensor map: sixteen cached tokens of a page, sixteen drafts (those that are none are
                // read by no row, and their values looked through; behind the last a map gives zeros), or, of values, no token at all.
                const int pos = tile * kTcTile + (lane & 7) * 16;
                int in = pos - (int)(p.page.div((uint32_t)pos) * p.page.d);
                const bool none = values && !draft && (p.boxes & 1) && pos >= at.len;
                const uint32_t nothing = __ballot_sync(0xffffffffu, none) & 0xffu;
                if (none) { page = 0; in = (int)p.page.d; }
                const bool whole16 = draft ? (p.boxes & 4) != 0 : none || ((p.boxes & 1) && pos + 16 <= at.len && page >= 0 && page < p.pages);
                const uint32_t boxes = __ballot_sync(0xffffffffu, whole16) & 0xffu;
                // others, row by row: which keys there are, and where (lane x the key x of each 32)
                uint32_t words[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
                unsigned long long rows[4];
                if (boxes != 0xffu) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const char *kk = p.q, *vv = p.q;
                        words[i] = __ballot_sync(0xffffffffu, key_row(p, Place{at.b, at.unit, tile, at.tiles, at.len}, kv, i * 32 + lane, kk, vv, &bad));
                        rows[i] = reinterpret_cast<unsigned long long>(values ? vv : kk);
                    }
                }
                wait(empty, ((uint32_t)turn & 1u) ^ 1u);
                if (lane < 4) {
                    if (values) spoilt[(t & 7) * 4 + lane] = 0;
                    else valid[(t & 7) * 4 + lane] = lane == 0 ? words[0] : lane == 1 ? words[1] : lane == 2 ? words[2] : words[3];
                }
                __syncwarp();
                // (a chain's drafts are read by all rows up to the first row's; others may hold anything, and are looked through)
                const bool look_through = values && draft && (p.parents || n0 + kTcTile - 1 > (int)p.group.div((uint32_t)row0));
                const int bar = look_through ? kRaw + cw : full;
                const uint32_t bytes = (uint32_t)__popc(boxes) * 256u * lanes;
                if (look_through || boxes == 0xffu) tell(bar, bytes);
                if (boxes) {
                    int pages[8], ins[8];
#pragma unroll
                    for (int sl = 0; sl < 8; ++sl) {
                        pages[sl] = __shfl_sync(0xffffffffu, page, sl);
                        ins[sl] = __shfl_sync(0xffffffffu, in, sl);
                    }
                    if (elect_one()) {
                        if (draft) {
#pragma unroll
                            for (int sl = 0; sl < 8; ++sl)
                                if (boxes >> sl & 1) box(values ? maps.dv : maps.dk, lanes / 8, bar, dst + sl * 2048, n0 + sl * 16, kv, at.b);
                        } else if (boxes == 0xffu && p.box_rows > 16 && !nothing) {
#pragma unroll
                            for (int sl = 0; sl < 8; sl += 2)
                                if (((sl * 16) & (p.box_rows - 1)) == 0) box(values ? maps.vb : maps.kb, lanes / 8, bar, dst + sl * 2048, ins[sl], kv, pages[sl]);
                        } else {
#pragma unroll
                            for (int sl = 0; sl < 8; ++sl)
                                if (boxes >> sl & 1) box(values ? maps.v : maps.k, lanes / 8, bar, dst + sl * 2048, ins[sl], kv, pages[sl]);
                        }
                    }
                    __syncwarp();
                }
                if (boxes != 0xffu) {
                    if (lanes == 16) copy_rows(std::integral_constant<int, 16>{}, dst, rows, words, boxes, width, values);
                    else copy_rows(std::integral_constant<int, 8>{}, dst, rows, words, boxes, width, values);
                    cp_async_commit();
                    if (values) cp_async_wait<0>();
                }
                // Rows of keys are told one tile later, when they have had time to come (their stage's next use is two tiles away; that of
                // values waits for them), while whole tiles of tokens follow.
                if (late_bar >= 0) {
                    if (boxes != 0xffu) cp_async_wait<1>(); else cp_async_wait<0>();
                    fence_proxy_async();
                    __syncwarp();
                    tell(late_bar, late_bytes);
                    late_bar = -1;
                }
                if (look_through) {
                    wait(bar, raws++ & 1u);
                    __syncwarp();
                    const int rows_in = min(p.N - n0, kTcTile);
#pragma unroll 2
                    for (int x = lane; x < rows_in * lanes; x += 32)
                        if (take_out<T>(dst + place_of(x / lanes, x % lanes))) atomicOr(&spoilt[(t & 7) * 4 + (x / lanes >> 5)], 1u << (x / lanes & 31));
                }
                if (!values && boxes != 0xffu && j + 1 < piece && (tile + 2) * kTcTile <= at.len) {
                    late_bar = full;
                    late_bytes = bytes;
                } else if (look_through || boxes != 0xffu) {
                    if (!values) cp_async_wait<0>();
                    fence_proxy_async();
                    __syncwarp();
                    tell(full, look_through ? 0 : bytes);
                }
                if (j + jstep < piece) look(tile + jstep);
                last = t;
            }
            if (late_bar >= 0) {
                cp_async_wait<0>();
                fence_proxy_async();
                __syncwarp();
                tell(late_bar, late_bytes);
            }
            g += piece;
            done += share;
            ++unit_no;
            at.tile += share - 1;
            at.next(p);
        }
        if (last >= 0) {                                  // whatever happened: nothing is in flight when the block ends
            if (cw > 0) late |= !mbar_wait_bounded(bars + kVFull + last % VS, (uint32_t)(last / VS) & 1u, kTcWaitCap);
            else late |= !mbar_wait_bounded(bars + kKFull + last % KS, (uint32_t)(last / KS) & 1u, kTcWaitCap);
        }
    } else if (w == kTcMma) {
        // ---- products
        if (elect_one()) {
            const uint32_t base = smem_u32(sm), iqk = tc_idesc(BF, p.neg, false, kTcTile), ipv = tc_idesc(BF, false, true, DV);
            auto qk = [&](int half, int rows, int st) {
                const uint32_t a = tc_desc(base + S::q + rows * S::qhalf, 16), b = tc_desc(base + S::k + st * S::kst, 16);
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks) {
                    const uint32_t off = ((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4;
                    tc_mma_ss(tmem + half * 128, a + off, b + off, iqk, ks > 0);
                }
            };
            auto pv = [&](int half, int st) {
                const uint32_t b = tc_desc(base + S::v + st * S::vst, 128 * 128);
#pragma unroll
                for (int ks = 0; ks < kTcTile / 16; ++ks) tc_mma_ts(tmem + 256 + half * 128, tmem + half * 128 + ks * 8, b + ks * (2048 >> 4), ipv);
            };
            int g = 0, unit_no = 0, done = 0;
            uint32_t had[2] = {0, 0};                     // jobs whose P a half has had
            while (done < n_tiles) {
                const int share = min(n_tiles - done, at.tiles - at.tile), piece = useful(at, share);
                if (piece == 0) {
                    done += share;
                    at.tile += share - 1;
                    at.next(p);
                    continue;
                }
                // job i: half i & 1, tile i / 2 of the unit or (few rows) tile i
                const int two = two_halves(at) ? 1 : 0, jobs = piece << two;
                auto scores = [&](int i) {
                    const int t = g + (i >> two), st = t % KS;
                    if (!two || !(i & 1)) {
                        wait(kKFull + st, (uint32_t)(t / KS) & 1u);
                        tc_fence_after();
                    }
                    qk(i & 1, two ? i & 1 : 0, st);
                    tc_commit(bars + kSFull + (i & 1));
                    if (!two || (i & 1)) tc_commit(bars + kKEmpty + st);
                };
                wait(kQFull, unit_no & 1);
                scores(0);
                if (jobs > 1) scores(1);
                if (jobs <= 2) tc_commit(bars + kQEmpty);
                for (int i = 0; i < jobs; ++i) {
                    const int half = i & 1, t = g + (i >> two), st = t % VS;
                    if (!two || !half) wait(kVFull + st, (uint32_t)(t / VS) & 1u);
                    wait(kPReady + half, (half ? had[1]++ : had[0]++) & 1u);
                    tc_fence_after();
                    pv(half, st);
                    if (i + 2 >= jobs) tc_commit(bars + kOFull + half);
                    if (!two || half) tc_commit(bars + kVEmpty + st);
                    if (i + 2 < jobs) scores(i + 2);
                    if (i + 3 == jobs) tc_commit(bars + kQEmpty);
                }
                g += piece;
                done += share;
                ++unit_no;
                at.tile += share - 1;
                at.next(p);
            }
            tc_commit(bars + kDone);
            late |= !mbar_wait_bounded(bars + kDone, 0, kTcWaitCap);          // all products are done
        }
        __syncwarp();
    } else {
        // ---- softmax: a thread a row
        const int half = w >> 2, lane_row = (w & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)(w & 3) << 21;   // lane 32 * (w & 3) of tensor memory
        const uint32_t ts = tmem + lanes + half * 128, to = tmem + lanes + 256 + half * 128, to_other = tmem + lanes + 256 + (half ^ 1) * 128;
        float2* swap = reinterpret_cast<float2*>(sm + S::swap) + lane_row;   // reference and mass of a row, of one half at a time
        int g = 0, done = 0;
        uint32_t turns = 0, ends[2] = {0, 0};             // jobs of this half; units that either half had jobs of
        bool first_piece = true;
        while (done < n_tiles) {
            const int share = min(n_tiles - done, at.tiles - at.tile), piece = useful(at, share), cached = at.tiles - p.draft_tiles;
            const bool whole = at.tile == 0 && share == at.tiles, two = two_halves(at);
            if (tid == 0 && at.tile == 0) leave_task(p, at, x0 + done, x0, blockIdx.x, line, whole);
            const int row = two ? half * 128 + lane_row : lane_row, jobs = two ? piece : (piece + 1 - half) >> 1;
            int n, h;
            const bool on = row_of(p, at.unit, row, n, h);
            uint32_t x[2][16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[0][i] = 0;
#pragma unroll
            for (int c = 0; c < DV; c += 16) tc_st16(to + c, x[0]);
            float ref = 0.f, mass = 0.f;
            bool empty = true;                            // the row has had no key yet
            for (int i = 0; i < jobs; ++i) {
                const int j = two ? i : 2 * i + half, tile = at.tile + j, gg = g + j;
                wait(kSFull + half, turns++ & 1u);
                tc_fence_after();
                tc_ld16(x[0], ts);
                uint32_t seen[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) seen[c] = valid[(gg & 7) * 4 + c];
                if (tile >= cached) {
                    const int tile0 = (tile - cached) * kTcTile;
                    uint64_t own[2] = {0, 0};
                    if (on) draft_masks(p, at.b, n, tile0, own, &bad);
                    seen[0] &= (uint32_t)own[0]; seen[1] &= (uint32_t)(own[0] >> 32); seen[2] &= (uint32_t)own[1]; seen[3] &= (uint32_t)(own[1] >> 32);
                }
                uint32_t pk[64];
                float2 sums[2];
                sums[0] = sums[1] = make_float2(0.f, 0.f);
                // (A row whose scores are NaN, as those of padding may be, stays so and does not call for a new reference: that its neighbours'
                // would move with.)  P and its sum, of 16 scores; `mixed`: every kTcPolyEvery-th pair of exponentials on the FMA pipes, of which `high`
                // has the largest exponent
                float high = 0.f;
                auto weigh = [&](const uint32_t (&y)[16], uint32_t* to_pk, auto mixed) {
                    const float2 cc = make_float2(p.c, p.c), bb = make_float2(-ref, -ref);
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float2 t = ffma2(make_float2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), cc, bb);
                        const float2 v = decltype(mixed)::value && (e >> 1) % kTcPolyEvery == kTcPolyEvery - 1 ? exp2_poly(t, high) : make_float2(ex2_approx(t.x), ex2_approx(t.y));
                        sums[(e >> 1) & 1] = fadd2(sums[(e >> 1) & 1], v);
                        to_pk[e >> 1] = Frag<T>::pack(v.x, v.y);
                    }
                };
                bool anew = __any_sync(0xffffffffu, (seen[0] & seen[1] & seen[2] & seen[3]) != 0xffffffffu);
                if (!anew && __any_sync(0xffffffffu, empty && mass == mass)) {
                    // a first reference: the largest of sixteen scores (none is above the one that the maximum would give)
                    tc_wait_ld(x[0]);
                    float t = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 16; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(t) : "f"(__uint_as_float(x[0][e])));
                    if (empty && fabsf(t) <= 3.4028234e38f) {
                        ref = t * p.c - kTcBias<T>;
                        empty = false;
                    }
                    anew = __any_sync(0xffffffffu, empty && fabsf(t) > 3.4028234e38f);
                }
                if (!anew) {
                    // the reference stays, unless the weights get too large for the type: their sum tells (none is larger than it), and `high`
                    // where the sum means nothing
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        tc_wait_ld(x[c & 1]);
                        if (c < 7) tc_ld16(x[(c + 1) & 1], ts + (c + 1) * 16);
                        weigh(x[c & 1], pk + c * 8, std::true_type{});
                    }
                    anew = __any_sync(0xffffffffu, (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y) > kTcMost<T> || high > kPolyMost);
                    sums[0].x = fmaf(high, 0.f, sums[0].x);        // (NaN among them stays NaN)
                } else {
                    tc_wait_ld(x[0]);
                }
                if (anew) {
                    // the row's maximum first; the sums follow the reference if it moves
                    float top = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        tc_ld16(x[0], ts + c * 32);
                        tc_ld16(x[1], ts + c * 32 + 16);
                        tc_wait_ld(x[0]);
                        tc_wait_ld(x[1]);
                        const uint32_t there = c == 0 ? seen[0] : c == 1 ? seen[1] : c == 2 ? seen[2] : seen[3];
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            t0 = fmaxf(t0, (there >> e & 1) ? __uint_as_float(x[0][e]) : -INFINITY);
                            t1 = fmaxf(t1, (there >> (16 + e) & 1) ? __uint_as_float(x[1][e]) : -INFINITY);
                        }
                        top = fmaxf(top, fmaxf(t0, t1));
                    }
                    // (a row that has had nothing yet keeps a reference of zero, which is worth nothing)
                    const float want = top * p.c - kTcBias<T>, now = top == -INFINITY ? ref : empty ? want : fmaxf(ref, want);
                    const float keep = empty ? 1.f : ex2_approx(ref - now);
                    if (top != -INFINITY) empty = false;
                    ref = now;
                    mass *= keep;
                    if (__any_sync(0xffffffffu, keep != 1.f)) {
#pragma unroll 1
                        for (int c = 0; c < DV; c += 16) {
                            tc_ld16(x[0], to + c);
                            tc_wait_ld(x[0]);
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[0][e] = __float_as_uint(__uint_as_float(x[0][e]) * keep);
                            tc_st16(to + c, x[0]);
                        }
                    }
                    // (weights over 32 scores take the place of sixteen: never of scores still to be read)
                    sums[0] = sums[1] = make_float2(0.f, 0.f);
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        tc_ld16(x[0], ts + c * 32);
                        tc_ld16(x[1], ts + c * 32 + 16);
                        tc_wait_ld(x[0]);
                        tc_wait_ld(x[1]);
                        const uint32_t there = c == 0 ? seen[0] : c == 1 ? seen[1] : c == 2 ? seen[2] : seen[3];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[i][e] = (there >> (16 * i + e) & 1) ? x[i][e] : 0xff800000u;
                            weigh(x[i], pk + 8 * i, std::false_type{});
                        }
                        tc_st16(ts + c * 16, pk);
                    }
                } else {
                    tc_st32(ts, pk);
                    tc_st32(ts + 32, pk + 32);
                }
                if (tile >= cached) {
                    // values that are not finite, of drafts that this row reads
                    const int tile0 = (tile - cached) * kTcTile;
                    wait(kVFull + gg % VS, (uint32_t)(gg / VS) & 1u);
                    const uint32_t* sp = spoilt + (gg & 7) * 4;
                    if (sp[0] | sp[1] | sp[2] | sp[3]) {
                        tc_wait_st();
                        const char* v0 = p.v + at.b * p.v_b + head_of(p, at.unit) * p.v_h;
#pragma unroll 1
                        for (int key = 0; key < kTcTile; ++key) {
                            if (!(sp[key >> 5] >> (key & 31) & 1)) continue;
                            const uint32_t mine = key < 32 ? seen[0] : key < 64 ? seen[1] : key < 96 ? seen[2] : seen[3];
#pragma unroll 1
                            for (int c = 0; c < DV; c += 16) {
                                tc_ld16(x[0], to + c);
                                tc_wait_ld(x[0]);
                                if (mine >> (key & 31) & 1)
#pragma unroll
                                    for (int e = 0; e < 16; ++e)
                                        if (c + e < p.V) x[0][e] = __float_as_uint(put_back<T>(__uint_as_float(x[0][e]), v0 + (int64_t)(tile0 + key) * p.v_n, c + e));
                                tc_st16(to + c, x[0]);
                                tc_wait_st();
                            }
                        }
                    }
                }
                mass += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                tc_wait_st();
                tc_fence_before();
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bars + kPReady + half)) : "memory");
            }
            // with both halves on the same rows: one reference, the other half's sums added, each half for half the columns
            float f_own = 1.f, f_other = 0.f;
            int c0 = 0, c1 = DV;
            if (!two) {
                tc_wait_st();                             // (a half without jobs: its zeros)
                tc_fence_before();
                float2 other;
                const float2 mine = make_float2(empty ? -INFINITY : ref, mass);
                if (half == 0) *swap = mine;
                asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
                if (half == 1) { other = *swap; *swap = mine; }
                asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
                if (half == 0) other = *swap;
                const float own = empty ? -INFINITY : ref, t = fmaxf(own, other.x);
                if (t != -INFINITY) {
                    f_own = ex2_approx(own - t);
                    f_other = ex2_approx(other.x - t);
                    ref = t;
                    empty = false;
                }
                mass = mass * f_own + other.y * f_other;
                c0 = half * (DV / 2);
                c1 = c0 + DV / 2;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool had_any = piece > 0 && (two || i == 0 || piece > 1);
                if (had_any) {
                    if (!two || i == half) wait(kOFull + i, ends[i] & 1u);
                    ++ends[i];
                }
            }
            if (piece == 0) tc_wait_st();
            tc_fence_after();
            const bool real = on && is_draft(p, at.b, n), add = !two;
            const float inv = whole ? (real ? finish_scale(mass) : 0.f) : 1.f;
            const int64_t at_out = ((int64_t)at.b * p.N + n) * p.H + h;
            float* slot = p.part + (int64_t)(2 * blockIdx.x + (first_piece ? 0 : 1)) * p.rows * (p.V + 2);
            auto write = [&](const float (&o)[8], int col) {
                if (!on || col >= p.V) return;
                if (whole) {
                    uint4 y = make_uint4(Frag<T>::pack(o[0], o[1]), Frag<T>::pack(o[2], o[3]), Frag<T>::pack(o[4], o[5]), Frag<T>::pack(o[6], o[7]));
                    if (!real) y = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + at_out * p.V + col) = y;
                } else {
                    *reinterpret_cast<float4*>(slot + row * p.V + col) = make_float4(o[0], o[1], o[2], o[3]);
                    *reinterpret_cast<float4*>(slot + row * p.V + col + 4) = make_float4(o[4], o[5], o[6], o[7]);
                }
            };
            f_own *= inv;
            f_other *= inv;
#pragma unroll 1
            for (int c = c0; c < c1; c += add ? 16 : 32) {       // the sums of both halves, or 32 columns of this one's
                tc_ld16(x[0], to + c);
                tc_ld16(x[1], add ? to_other + c : to + c + 16);
                tc_wait_ld(x[0]);
                tc_wait_ld(x[1]);
                if (add) {
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        float o[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(x[0][i + e]) * f_own + __uint_as_float(x[1][i + e]) * f_other;
                        write(o, c + i);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float o[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(x[i >> 4][(i & 15) + e]) * f_own;
                        write(o, c + i);
                    }
                }
            }
            if (on && (two || half == 0)) {
                if (!whole) *reinterpret_cast<float2*>(slot + p.rows * p.V + 2 * row) = make_float2(empty ? -INFINITY : ref, mass);
                else if (p.lse) p.lse[at_out] = real ? finish_lse(ref, mass) : -INFINITY;
            }
            if (!two) {                                   // the other half has read this one's O, and this thread's words
                tc_fence_before();
                asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
                tc_fence_after();
            }
            g += piece;
            first_piece = false;
            done += share;
            at.tile += share - 1;
            at.next(p);
        }
        tc_fence_before();
    }
    __syncthreads();
    if (w == kTcMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    }
    if (p.status) {
        if (bad) atomicOr(p.status, HTREE_STATUS_CACHE);
        if (late) atomicOr(p.status, 16);
    }
}

// ---- joining the parts -------------------------------------------------------------------------------------------------------

// A task is the rows of a unit that several parts have left; by unit, or, where there are more units than parts, by the part that starts and
// does not finish it.  A team of 1 to 8 warps joins a row (as many parts as a unit has on average, about four to a warp), four parts in
// flight at a time.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
template <typename T, bool Wide>
__global__ void __launch_bounds__(kJoinThreads) draft_join_kernel(const __grid_constant__ DraftParams p) {
    constexpr int C = Wide ? 2 : 1;                      // columns lane*4 (and + 128)
    __shared__ float4 red[kJoinWarps][C][32];
    __shared__ float2 stat[kJoinWarps];
    chain_enter();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, team = w / p.team, member = w - team * p.team;
    const int4 task = p.tasks[blockIdx.x];
    if (task.x < 0) return;
    const int slots = task.w >> 1, r = blockIdx.y * (kJoinWarps / p.team) + team;
    const int64_t size = (int64_t)p.rows * (p.V + 2);
    int n = 0, h = 0;
    const bool on = r < p.rows && row_of(p, task.y, r, n, h);
    const bool real = on && is_draft(p, task.x, n);
    float top = -INFINITY, mass = 0.f;
    float4 o[C];
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
        const float* slot0 = p.part + 2 * (int64_t)task.z * size;
        for (int i0 = member; i0 < slots; i0 += 4 * p.team) {
            float2 rm[4];
            float4 x[4][C];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * p.team;
                rm[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int c = 0; c < C; ++c) x[u][c] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < slots) {
                    const float* s = slot0 + (i > 0 ? 2 * i * size : (task.w & 1) ? size : 0);
                    rm[u] = *reinterpret_cast<const float2*>(s + p.rows * p.V + 2 * r);
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        if (c * 128 + lane * 4 < p.V) x[u][c] = *reinterpret_cast<const float4*>(s + r * p.V + c * 128 + lane * 4);
                }
            }
            const float now = fmaxf(fmaxf(top, fmaxf(rm[0].x, rm[1].x)), fmaxf(rm[2].x, rm[3].x)), ref = now == -INFINITY ? 0.f : now;
            const float keep = exp2f(top - ref);
            top = now;
            mass *= keep;
#pragma unroll
            for (int c = 0; c < C; ++c) o[c] = make_float4(o[c].x * keep, o[c].y * keep, o[c].z * keep, o[c].w * keep);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float f = exp2f(rm[u].x - ref);
                mass = fmaf(f, rm[u].y, mass);
#pragma unroll
                for (int c = 0; c < C; ++c)
                    o[c] = make_float4(fmaf(f, x[u][c].x, o[c].x), fmaf(f, x[u][c].y, o[c].y), fmaf(f, x[u][c].z, o[c].z), fmaf(f, x[u][c].w, o[c].w));
            }
        }
    }
    if (p.team > 1) {
#pragma unroll
        for (int c = 0; c < C; ++c) red[w][c][lane] = o[c];
        if (lane == 0) stat[w] = make_float2(top, mass);
        __syncthreads();
        if (member > 0) return;
        float now = top;
        for (int i = 1; i < p.team; ++i) now = fmaxf(now, stat[w + i].x);
        const float ref = now == -INFINITY ? 0.f : now;
        mass = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < p.team; ++i) {
            const float f = exp2f(stat[w + i].x - ref);
            mass = fmaf(f, stat[w + i].y, mass);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float4 x = red[w + i][c][lane];
                o[c] = make_float4(fmaf(f, x.x, o[c].x), fmaf(f, x.y, o[c].y), fmaf(f, x.z, o[c].z), fmaf(f, x.w, o[c].w));
            }
        }
        top = now;
    }
    if (!on) return;
    const int64_t row = ((int64_t)task.x * p.N + n) * p.H + h;
    const float inv = real ? finish_scale(mass) : 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int col = c * 128 + lane * 4;
        if (col >= p.V) continue;
        T* to = reinterpret_cast<T*>(p.out) + row * p.V + col;
        const float4 y = real ? make_float4(o[c].x * inv, o[c].y * inv, o[c].z * inv, o[c].w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = y;
        else *reinterpret_cast<uint2*>(to) = make_uint2(Frag<T>::pack(y.x, y.y), Frag<T>::pack(y.z, y.w));
    }
    if (p.lse && lane == 0) p.lse[row] = real ? finish_lse(top, mass) : -INFINITY;
}

// ---- launches ----------------------------------------------------------------------------------------------------------------

static int64_t units_of(const DraftParams& p) { return (int64_t)p.B * p.Hkv * p.row_tiles; }

// least: tiles that a part has at least (a block's warps, each of which takes one at a time).
static void fit(DraftParams& p, int rows, int tile, int blocks, int least) {
    p.rows = rows;
    p.row_tiles = (p.N * p.G + rows - 1) / rows;
    p.per_head = FastDiv((uint32_t)p.row_tiles);
    p.shift = tile == 16 ? 4 : tile == 64 ? 6 : 7;
    p.draft_tiles = (p.N + tile - 1) / tile;
    p.grid = blocks;
    p.least = least;
    // With tables so short that a block is done with any unit in two rounds of its warps (tcgen05: in four tiles), parts are whole units, and
    // the second kernel, 4 of 15 us of a small call, falls away.
    const int most = ((p.room + tile - 1) >> p.shift) + p.draft_tiles;
    p.whole = most <= (tile == kSlice ? 2 * least : 4);
    if (p.whole && units_of(p) < p.grid) p.grid = (int32_t)units_of(p);
    p.by_unit = units_of(p) <= p.grid;
    const int64_t each = p.grid / units_of(p);         // parts of a unit
    p.team = each >= 16 ? 8 : each >= 8 ? 4 : each >= 4 ? 2 : 1;
}
static int64_t part_bytes(const DraftParams& p) { return p.whole ? 0 : (int64_t)p.grid * 2 * p.rows * (p.V + 2) * 4; }
static int64_t workspace_of(const DraftParams& p) { return p.whole ? 16 : part_bytes(p) + p.grid * 16; }           // tasks: per unit or per part, never more than parts

// Which kernel.  16-bit rows of up to 128 go to the tensor cores, by mma.sync up to 32 query rows, up to 16 with rows of more than 64 (where
// a warp of 32 has spills).  Measured, 8 requests of 16384, 4 heads of 128: 32 rows 104 us on mma.sync (two tiles of sixteen) and 63 on
// tcgen05, 16 rows 63 and 62; 8 heads of 64: 32 rows 76 and 80; 8 requests of 1000, 4 heads of 128: 32 rows 23.4 and 20.4, 16 rows 18.5 and 19.4.
// fp32 (4 requests of 16384, 4 heads of 128): 17 to 32 rows 266 us by slices of sixteen rows and 242 by FFMA tiles of 64, 16 rows 147 and
// 242; 8 rows 95 by slices of eight and 148 by those of sixteen.  Wider 16-bit rows: slices of 16 query rows however many there are (4 requests of 16384, 4 heads of 256, 256 rows: 620 us).
enum { kSlice4 = 0, kSlice8, kSlice16, kSlice32, kFma, kTc };
static void choose(DraftParams& p, int dtype) {
    const int sms = sm_count() > 0 ? sm_count() : 148, rows = p.N * p.G;
    const bool wide = p.K > 128 || p.V > 128;
    if (dtype == HTREE_F32) {
        p.variant = rows <= 4 ? kSlice4 : rows <= 8 ? kSlice8 : rows <= 16 ? kSlice16 : kFma;
        if (p.variant == kFma) fit(p, kFmaRows, kTile, wide ? sms : 2 * sms, 1);
        else fit(p, rows <= 4 ? 4 : rows <= 8 ? 8 : 16, kSlice, sms, wide ? 3 : p.K > 64 && p.V > 64 ? 6 : p.K > 64 || p.V > 64 ? 8 : 12);
        return;
    }
    p.variant = wide || rows <= 16 ? kSlice16 : rows <= 32 && p.K <= 64 && p.V <= 64 ? kSlice32 : kTc;
    if (p.variant == kTc) fit(p, rows <= 128 ? 128 : 256, kTcTile, sms, 1);
    else fit(p, p.variant == kSlice16 ? 16 : 32, kSlice, sms, wide ? 6 : p.variant == kSlice16 ? 12 : 8);
    if (p.c < 0.f) { p.neg = 1; p.c = -p.c; }
    if (p.c < 1.1754944e-38f) p.c = 1.1754944e-38f;        // a scale of zero: scores of zero, but what is masked stays minus infinity
}

// A tensor map over three dimensions of rows; false where the strides are none that a map can have (an expanded dimension), or the driver has
// no such call.
struct MapDim { int64_t size, stride; uint32_t box; };
static bool row_map(CUtensorMap& map, const char* base, int width, const MapDim (&d)[3], bool bf16) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<Encode>(f);
    }();
    cuuint64_t dims[4] = {(cuuint64_t)width, 0, 0, 0}, strides[3];
    cuuint32_t box[4] = {64, 0, 0, 0};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = (cuuint64_t)d[i].size;
        strides[i] = (cuuint64_t)(d[i].size > 1 ? d[i].stride : 16);       // (of one element it is never used, but has to be one)
        box[i + 1] = d[i].box;
        if (strides[i] == 0 || strides[i] >= (cuuint64_t(1) << 40) || dims[i + 1] > (cuuint64_t(1) << 32) || box[i + 1] > 256) return false;
    }
    return encode && encode(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<char*>(base), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static int tc_maps(TcMaps& m, DraftParams& p, bool bf16) {
    int boxes = 0;
    auto caches = [&](CUtensorMap& k, CUtensorMap& v, uint32_t rows) {
        return row_map(k, p.ck, p.K, {{(int64_t)p.page.d, p.ck_row, rows}, {p.Hkv, p.ck_h, 1}, {p.pages, p.ck_page, 1}}, bf16) &&
               row_map(v, p.cv, p.V, {{(int64_t)p.page.d, p.cv_row, rows}, {p.Hkv, p.cv_h, 1}, {p.pages, p.cv_page, 1}}, bf16);
    };
    p.box_rows = p.page.d % 128 == 0 ? 128 : p.page.d % 64 == 0 ? 64 : p.page.d % 32 == 0 ? 32 : 16;
    if (p.page.d % 16 == 0 && caches(m.k, m.v, 16)) boxes |= 1;
    if (p.box_rows > 16 && !caches(m.kb, m.vb, (uint32_t)p.box_rows)) p.box_rows = 16;
    if (128 % p.G == 0 && row_map(m.q, p.q, p.K, {{p.H, p.q_h, (uint32_t)p.G}, {p.N, p.q_n, (uint32_t)(128 / p.G)}, {p.B, p.q_b, 1}}, bf16)) boxes |= 2;
    if (row_map(m.dk, p.k, p.K, {{p.N, p.k_n, 16}, {p.Hkv, p.k_h, 1}, {p.B, p.k_b, 1}}, bf16) &&
        row_map(m.dv, p.v, p.V, {{p.N, p.v_n, 16}, {p.Hkv, p.v_h, 1}, {p.B, p.v_b, 1}}, bf16))
        boxes |= 4;
    return boxes;
}

template <typename T, int DK, int DV, int ROWS>
static int launch_slices(const DraftParams& p, cudaStream_t st) {
    static SmemLimit limit;
    using S = SliceShape<T, DK, DV, ROWS>;
    if (const cudaError_t e = limit.raise((const void*)draft_slice_kernel<T, DK, DV, ROWS>, S::total)) return (int)e;
    return launch_chained(draft_slice_kernel<T, DK, DV, ROWS>, dim3(p.grid), dim3(S::threads), S::total, st, p);
}
template <typename T, int DK, int DV>
static int launch_sized(const DraftParams& p, cudaStream_t st) {
    if constexpr (sizeof(T) == 4) {
        return p.variant == kSlice4 ? launch_slices<T, DK, DV, 4>(p, st) : p.variant == kSlice8 ? launch_slices<T, DK, DV, 8>(p, st) : launch_slices<T, DK, DV, 16>(p, st);
    } else {
    if constexpr (DK <= 128)
    if (p.variant == kTc) {
        static SmemLimit limit;
        if (const cudaError_t e = limit.raise((const void*)draft_tc_kernel<T, DK, DV>, TcShape<DK, DV>::total)) return (int)e;
        TcMaps maps{};
        DraftParams q = p;
        q.boxes = tc_maps(maps, q, std::is_same<T, __nv_bfloat16>::value);
        return launch_chained(draft_tc_kernel<T, DK, DV>, dim3(p.grid), dim3(kTcThreads), TcShape<DK, DV>::total, st, q, maps);
    }
    if constexpr (DK == 64 && DV == 64)
        if (p.variant == kSlice32) return launch_slices<T, DK, DV, 32>(p, st);
    return launch_slices<T, DK, DV, 16>(p, st);
    }
}

template <int D>
static int launch_fma(const DraftParams& p, cudaStream_t st) {
    static SmemLimit limit;
    if (const cudaError_t e = limit.raise((const void*)draft_fma_kernel<D>, FmaShape<D>::total)) return (int)e;
    return launch_chained(draft_fma_kernel<D>, dim3(p.grid), dim3(kFmaThreads), FmaShape<D>::total, st, p);
}

template <typename T>
static int launch_draft(const DraftParams& p, cudaStream_t st) {
    const bool k64 = p.K <= 64, v64 = p.V <= 64;
    int rc;
    if (p.variant == kFma) rc = k64 && v64 ? launch_fma<64>(p, st) : p.K <= 128 && p.V <= 128 ? launch_fma<128>(p, st) : launch_fma<256>(p, st);
    else if (p.K > 128 || p.V > 128) rc = launch_sized<T, 256, 256>(p, st);
    else rc = k64 ? (v64 ? launch_sized<T, 64, 64>(p, st) : launch_sized<T, 64, 128>(p, st)) : v64 ? launch_sized<T, 128, 64>(p, st) : launch_sized<T, 128, 128>(p, st);
    if (rc || p.whole) return rc;
    const int rows = p.N * p.G < p.rows ? p.N * p.G : p.rows, block = kJoinWarps / p.team;
    const dim3 grid(p.by_unit ? (unsigned)units_of(p) : (unsigned)p.grid, (rows + block - 1) / block);
    return p.V > 128 ? launch_chained(draft_join_kernel<T, true>, grid, dim3(kJoinThreads), 0, st, p)
                     : launch_chained(draft_join_kernel<T, false>, grid, dim3(kJoinThreads), 0, st, p);
}

static int fill_draft(DraftParams& p, const HtreeCache* c, const HtreeDrafts* d) {
    if (const int rc = check_cache(c)) return rc;
    if (!d) return HTREE_E_NULL;
    if (d->B <= 0 || d->N <= 0 || d->H <= 0 || d->M <= 0 || d->H % c->H_kv != 0 || d->table_stride < d->M) return HTREE_E_SHAPE;
    const int64_t rows = (int64_t)d->N * (d->H / c->H_kv);
    if (c->K > 256 || c->V > 256 || (d->parents && d->N > kMaxTree) || rows > (1 << 24) || c->page_size > (1 << 20)) return HTREE_E_UNSUPPORTED;
    if ((int64_t)d->B * c->H_kv * rows >= (int64_t(1) << 31)) return HTREE_E_UNSUPPORTED;
    const int es = cache_esize(c->dtype);
    p = DraftParams{};
    p.q = (const char*)d->q; p.k = (const char*)d->k; p.v = (const char*)d->v; p.ck = (const char*)c->k; p.cv = (const char*)c->v;
    p.table = d->table; p.lengths = d->lengths; p.parents = d->parents; p.out = d->out; p.lse = d->lse;
    p.q_b = d->q_stride[0] * es; p.q_n = d->q_stride[1] * es; p.q_h = d->q_stride[2] * es;
    p.k_b = d->k_stride[0] * es; p.k_n = d->k_stride[1] * es; p.k_h = d->k_stride[2] * es;
    p.v_b = d->v_stride[0] * es; p.v_n = d->v_stride[1] * es; p.v_h = d->v_stride[2] * es;
    p.ck_page = c->k_page * es; p.ck_row = c->k_row * es; p.ck_h = c->k_head * es;
    p.cv_page = c->v_page * es; p.cv_row = c->v_row * es; p.cv_h = c->v_head * es;
    p.table_stride = d->table_stride;
    p.B = d->B; p.N = d->N; p.H = d->H; p.Hkv = c->H_kv; p.G = d->H / c->H_kv; p.K = c->K; p.V = c->V; p.pages = c->pages;
    const int64_t room = (int64_t)d->M * c->page_size;
    p.room = (int32_t)(room < kMaxLength ? room : kMaxLength);
    if ((int64_t)d->B * ((p.room + kSlice - 1) / kSlice + (d->N + kSlice - 1) / kSlice) >= (int64_t(1) << 31)) return HTREE_E_UNSUPPORTED;
    p.c = d->scale * kLog2e;
    p.page = FastDiv((uint32_t)c->page_size);
    p.group = FastDiv((uint32_t)p.G);
    choose(p, c->dtype);
    return 0;
}

}  // namespace htree

using namespace htree;

extern "C" {

int64_t htree_b200_draft_workspace(const HtreeCache* cache, const HtreeDrafts* drafts) {
    DraftParams p;
    if (const int rc = fill_draft(p, cache, drafts)) return rc;
    return workspace_of(p);
}

int htree_b200_draft_attention(const HtreeCache* cache, const HtreeDrafts* drafts, void* workspace, int64_t workspace_bytes,
                               int32_t* status, void* stream) {
    DraftParams p;
    if (const int rc = fill_draft(p, cache, drafts)) return rc;
    if (!p.q || !p.k || !p.v || !p.table || !p.lengths || !p.out || !workspace) return HTREE_E_NULL;
    const int es = cache_esize(cache->dtype);
    if (!cache_aligned(p.q) || !cache_aligned(p.k) || !cache_aligned(p.v) || !cache_aligned(p.out) || !cache_aligned(workspace) ||
        !cache_strides_ok(drafts->q_stride, es) || !cache_strides_ok(drafts->k_stride, es) || !cache_strides_ok(drafts->v_stride, es))
        return HTREE_E_ALIGN;
    if (workspace_bytes < workspace_of(p)) return HTREE_E_SCRATCH;
    p.part = (float*)workspace;
    p.tasks = (int4*)((char*)workspace + part_bytes(p));
    p.status = status;
    const cudaStream_t st = (cudaStream_t)stream;
    return cache->dtype == HTREE_F32 ? launch_draft<float>(p, st)
         : cache->dtype == HTREE_BF16 ? launch_draft<__nv_bfloat16>(p, st) : launch_draft<__half>(p, st);
}

}  // extern "C"
