// Attention of drafted tokens over a paged cache and over the drafts that lead to them.
//
// Work: the query rows that share a key/value head (drafts x heads of the group) are cut into row tiles; a unit is a request, a key/value
// head and a row tile, and its keys are tiles of 64: the cached tokens first, then the drafts.  All tiles of all units stand in one line
// that is cut into equal parts, one per block, whatever the lengths (which only the device knows).  A unit that lies in one part is
// finished there; of the others every part leaves its unnormalised sum, its maximum and its mass, which a second kernel joins in the order
// of the parts: the result does not depend on timing.
#include "cache.cuh"
#include "mma_common.cuh"

namespace htree {

constexpr int kTile = 64;                 // keys of a tile
constexpr int kMaxTree = 1024;
constexpr int64_t kMaxLength = int64_t(1) << 30;

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
    float* part;              // per slot: rows x V sums, then rows x {maximum, mass}; slots 2c and 2c+1 are block c's first and last unit
    int32_t* status;
    int64_t q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h;                  // strides in bytes
    int64_t ck_page, ck_row, ck_h, cv_page, cv_row, cv_h;
    int64_t table_stride;
    int32_t B, N, H, Hkv, G, K, V, M, pages;
    int32_t rows, row_tiles, draft_tiles, grid;                            // rows of a tile
    int32_t variant;          // which kernel (choose)
    int32_t neg;              // tensor-core kernels: the scale is negative, c its magnitude and q's signs are turned
    float c;                  // scale * log2 e
    FastDiv page, group;      // by G
};

// ---- the line of tiles -------------------------------------------------------------------------------------------------------

__device__ __forceinline__ int draft_length(const DraftParams& p, int b, bool* bad) {
    int64_t len = p.lengths[b], room = (int64_t)p.M * p.page.d;
    if (room > kMaxLength) room = kMaxLength;
    if (len < 0 || len > room) { *bad = true; len = len < 0 ? 0 : room; }
    return (int)len;
}
__device__ __forceinline__ int draft_tiles_of(const DraftParams& p, int b) {
    bool dull = false;
    return (draft_length(p, b, &dull) + kTile - 1) / kTile + p.draft_tiles;
}

// Where a part of the line is: request, unit of the request (head * row_tiles + row tile), tile of the unit.
struct Place {
    int b, unit, tile, tiles, len;
    __device__ __forceinline__ void enter(const DraftParams& p, int b_) {
        bool dull = false;
        b = b_;
        len = draft_length(p, b, &dull);
        tiles = (len + kTile - 1) / kTile + p.draft_tiles;
    }
    __device__ __forceinline__ void next(const DraftParams& p) {
        if (++tile < tiles) return;
        tile = 0;
        if (++unit < p.Hkv * p.row_tiles) return;
        unit = 0;
        if (b + 1 < p.B) enter(p, b + 1);
    }
};

// Blocks that take part, and where block c's part starts.
__device__ __forceinline__ int64_t parts_of(const DraftParams& p, int64_t all) { return all < p.grid ? all : p.grid; }
__device__ __forceinline__ int64_t part_start(int64_t c, int64_t all, int64_t parts) { return c * all / parts; }

// All tiles of the line (returned), and the place of tile x(all): every thread takes a stretch of requests, one scan over the block.
template <int NT, typename X>
__device__ __forceinline__ int64_t find_place(const DraftParams& p, X x, Place& at) {
    __shared__ int64_t scratch[NT / 32];
    __shared__ int64_t found[2];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, per = (p.B + NT - 1) / NT;
    const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B), units = p.Hkv * p.row_tiles;
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += draft_tiles_of(p, b);
    int64_t in = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += y;
    }
    if (lane == 31) scratch[w] = in;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int i = 0; i < NT / 32; ++i) {
        if (i < w) before += scratch[i];
        all += scratch[i];
    }
    all *= units;
    const int64_t want = x(all);
    before = (before + in - mine) * units;
    if (want >= before && want < before + mine * units) {
        int b = b0;
        int64_t t = draft_tiles_of(p, b);
        while (want >= before + t * units) { before += t * units; t = draft_tiles_of(p, ++b); }
        found[0] = b;
        found[1] = want - before;
    }
    __syncthreads();
    at.enter(p, (int)found[0]);
    at.unit = (int)(found[1] / at.tiles);
    at.tile = (int)(found[1] - (int64_t)at.unit * at.tiles);
    return all;
}

// Row r of a row tile: draft and head.  False behind the last row.
__device__ __forceinline__ bool row_of(const DraftParams& p, int unit, int r, int& n, int& h) {
    const int kv = unit / p.row_tiles, row = (unit - kv * p.row_tiles) * p.rows + r;
    n = (int)p.group.div((uint32_t)row);
    h = kv * p.G + row - n * p.G;
    return row < p.N * p.G;
}

// Which of the drafts tile0 .. tile0 + 63 draft n reads.
__device__ __forceinline__ uint64_t draft_mask(const DraftParams& p, int b, int n, int tile0, bool* bad) {
    if (!p.parents) {                                        // a chain: n and all before it
        const int upto = n - tile0;
        return upto < 0 ? 0ull : upto >= 63 ? ~0ull : (2ull << upto) - 1ull;
    }
    const int32_t* par = p.parents + (int64_t)b * p.N;
    if (par[n] < -1) return 0ull;
    uint64_t m = 0;
    for (int i = n; i >= tile0;) {                           // parents come before their children: at most n steps
        if (i < tile0 + 64) m |= 1ull << (i - tile0);
        const int up = par[i];
        if (up >= i) { *bad = true; break; }
        i = up;
    }
    return m;
}
__device__ __forceinline__ bool is_draft(const DraftParams& p, int b, int n) { return !p.parents || p.parents[(int64_t)b * p.N + n] >= -1; }

// Where the row of key j of a tile starts (keys, values); false for what the tile does not have.
__device__ __forceinline__ bool key_row(const DraftParams& p, const Place& at, int kv, int j, const char*& k, const char*& v, bool* bad) {
    const int cached = at.tiles - p.draft_tiles;
    if (at.tile < cached) {
        const int pos = at.tile * kTile + j;
        if (pos >= at.len) return false;
        const uint32_t i = p.page.div((uint32_t)pos);
        const int pg = __ldg(p.table + (int64_t)at.b * p.table_stride + i);
        if (pg < 0 || pg >= p.pages) { *bad = true; return false; }
        const int64_t in = (int64_t)(pos - i * p.page.d);
        k = p.ck + pg * p.ck_page + in * p.ck_row + kv * p.ck_h;
        v = p.cv + pg * p.cv_page + in * p.cv_row + kv * p.cv_h;
        return true;
    }
    const int n = (at.tile - cached) * kTile + j;
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

// ---- any type, any row width: fp32 arithmetic --------------------------------------------------------------------------------

// 16 rows a block, four a warp; a warp's scores stay in it: lane x holds keys x and x + 32, and the columns 4x .. 4x + 3 (and + 128) of
// the sums.
constexpr int kGenRows = 16, kGenThreads = 128;

template <typename T>
__device__ __forceinline__ void load8(const char* src, float* dst) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(src)), b = __ldg(reinterpret_cast<const float4*>(src) + 1);
        *reinterpret_cast<float4*>(dst) = a;
        *reinterpret_cast<float4*>(dst + 4) = b;
    } else {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(src));
        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Frag<T>::unpack(u[i]);
            dst[2 * i] = f.x;
            dst[2 * i + 1] = f.y;
        }
    }
}

template <typename T, int VC>
__global__ void __launch_bounds__(kGenThreads) draft_generic_kernel(const __grid_constant__ DraftParams p) {
    extern __shared__ __align__(16) float smem[];
    const int KS = p.K + 4, VS = VC * 128;
    float* sk = smem;                               // [64][KS]: four floats on a row of eight threads meet in no bank
    float* sv = sk + kTile * KS;                    // [64][VS], columns behind V zero
    float* sq = sv + kTile * VS;                    // [16][K]
    float* sp = sq + kGenRows * p.K;                // [16][64]
    __shared__ uint64_t mask[kGenRows];
    __shared__ uint8_t there[kTile];
    chain_enter();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    Place at;
    int64_t x0 = 0, x1 = 0;
    const int64_t all = find_place<kGenThreads>(p, [&](int64_t n) {
        const int64_t parts = parts_of(p, n);
        x0 = part_start(blockIdx.x < parts ? blockIdx.x : 0, n, parts);
        x1 = part_start(blockIdx.x < parts ? blockIdx.x + 1 : 1, n, parts);
        return x0;
    }, at);
    if (blockIdx.x >= parts_of(p, all)) return;
    bool bad = false;
    { bool b = false; draft_length(p, at.b, &b); bad |= b; }
    float m[4], mass[4], o[4][4 * VC];
    int first_tile = at.tile;                       // of the unit's part in this block
    bool fresh = true, first_piece = true;
    for (int64_t x = x0; x < x1; ++x) {
        const int kv = at.unit / p.row_tiles;
        if (fresh) {
            first_tile = at.tile;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                m[r] = -INFINITY;
                mass[r] = 0.f;
#pragma unroll
                for (int i = 0; i < 4 * VC; ++i) o[r][i] = 0.f;
            }
            __syncthreads();
            const int pieces = p.K / 8;
            for (int i = tid; i < kGenRows * pieces; i += kGenThreads) {
                const int r = i / pieces, c = i - r * pieces;
                int n, h;
                float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (row_of(p, at.unit, r, n, h)) load8<T>(p.q + at.b * p.q_b + n * p.q_n + h * p.q_h + c * 8 * (int)sizeof(T), f);
#pragma unroll
                for (int e = 0; e < 8; ++e) sq[r * p.K + c * 8 + e] = f[e];
            }
            fresh = false;
        }
        const bool draft = at.tile >= at.tiles - p.draft_tiles;
        __syncthreads();
        // two threads a key row
        {
            const int j = tid >> 1, half = tid & 1;
            const char *k = nullptr, *v = nullptr;
            const bool on = key_row(p, at, kv, j, k, v, &bad);
            if (half == 0) there[j] = on;
            for (int c = half; c < p.K / 8; c += 2) {
                float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (on) load8<T>(k + c * 8 * (int)sizeof(T), f);
                *reinterpret_cast<float4*>(sk + j * KS + c * 8) = make_float4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<float4*>(sk + j * KS + c * 8 + 4) = make_float4(f[4], f[5], f[6], f[7]);
            }
            for (int c = half; c < VS / 8; c += 2) {
                float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (on && c < p.V / 8) load8<T>(v + c * 8 * (int)sizeof(T), f);
                *reinterpret_cast<float4*>(sv + j * VS + c * 8) = make_float4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<float4*>(sv + j * VS + c * 8 + 4) = make_float4(f[4], f[5], f[6], f[7]);
            }
        }
        if (draft && tid < kGenRows) {
            int n, h;
            mask[tid] = row_of(p, at.unit, tid, n, h) ? draft_mask(p, at.b, n, (at.tile - (at.tiles - p.draft_tiles)) * kTile, &bad) : 0ull;
        }
        __syncthreads();
        float s[4][2];
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r][0] = s[r][1] = 0.f;
        for (int d = 0; d < p.K; d += 4) {
            const float4 a = *reinterpret_cast<const float4*>(sk + lane * KS + d), b = *reinterpret_cast<const float4*>(sk + (lane + 32) * KS + d);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 q = *reinterpret_cast<const float4*>(sq + (w * 4 + r) * p.K + d);
                s[r][0] = fmaf(q.w, a.w, fmaf(q.z, a.z, fmaf(q.y, a.y, fmaf(q.x, a.x, s[r][0]))));
                s[r][1] = fmaf(q.w, b.w, fmaf(q.z, b.z, fmaf(q.y, b.y, fmaf(q.x, b.x, s[r][1]))));
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint64_t seen = draft ? mask[w * 4 + r] : ~0ull;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = lane + 32 * i;
                s[r][i] = there[j] && (seen >> j & 1) ? s[r][i] * p.c : -INFINITY;
            }
            const float top = fmaxf(m[r], warp_max(fmaxf(s[r][0], s[r][1]))), ref = top == -INFINITY ? 0.f : top;
            const float keep = exp2f(m[r] - ref), e0 = exp2f(s[r][0] - ref), e1 = exp2f(s[r][1] - ref);
            m[r] = top;
            mass[r] = fmaf(mass[r], keep, e0 + e1);
#pragma unroll
            for (int i = 0; i < 4 * VC; ++i) o[r][i] *= keep;
            sp[(w * 4 + r) * kTile + lane] = e0;
            sp[(w * 4 + r) * kTile + lane + 32] = e1;
        }
        __syncwarp();
        for (int j = 0; j < kTile; j += 4) {
            float pr[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) *reinterpret_cast<float4*>(pr[r]) = *reinterpret_cast<const float4*>(sp + (w * 4 + r) * kTile + j);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(sv + (j + i) * VS + c * 128 + lane * 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (draft && !(mask[w * 4 + r] >> (j + i) & 1)) continue;      // a draft's values, whatever they are, stay with those that read it
                        o[r][4 * c] = fmaf(pr[r][i], v.x, o[r][4 * c]);
                        o[r][4 * c + 1] = fmaf(pr[r][i], v.y, o[r][4 * c + 1]);
                        o[r][4 * c + 2] = fmaf(pr[r][i], v.z, o[r][4 * c + 2]);
                        o[r][4 * c + 3] = fmaf(pr[r][i], v.w, o[r][4 * c + 3]);
                    }
                }
        }
        __syncwarp();
        const bool done = at.tile + 1 == at.tiles;
        if (done || x + 1 == x1) {                  // the unit ends, or this block's part of it
            const bool whole = done && first_tile == 0;
            float* slot = p.part + (int64_t)(2 * blockIdx.x + (first_piece ? 0 : 1)) * kGenRows * (p.V + 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float sum = warp_sum(mass[r]);
                int n, h;
                if (!row_of(p, at.unit, w * 4 + r, n, h)) continue;
                if (whole) {
                    const bool real = is_draft(p, at.b, n);
                    const float inv = real ? finish_scale(sum) : 0.f;
                    const int64_t row = ((int64_t)at.b * p.N + n) * p.H + h;
#pragma unroll
                    for (int i = 0; i < 4 * VC; ++i) {
                        const int c = (i / 4) * 128 + lane * 4 + (i & 3);
                        if (c < p.V) reinterpret_cast<T*>(p.out)[row * p.V + c] = from_f<T>(real ? o[r][i] * inv : 0.f);
                    }
                    if (p.lse && lane == 0) p.lse[row] = real ? finish_lse(m[r], sum) : -INFINITY;
                } else {
#pragma unroll
                    for (int i = 0; i < 4 * VC; ++i) {
                        const int c = (i / 4) * 128 + lane * 4 + (i & 3);
                        if (c < p.V) slot[(w * 4 + r) * p.V + c] = o[r][i];
                    }
                    if (lane == 0) {
                        slot[kGenRows * p.V + 2 * (w * 4 + r)] = m[r];
                        slot[kGenRows * p.V + 2 * (w * 4 + r) + 1] = sum;
                    }
                }
            }
            first_piece = false;
            fresh = true;
        }
        const int b = at.b;
        at.next(p);
        if (at.b != b) { bool d = false; draft_length(p, at.b, &d); bad |= d; }
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
}

// ---- 16-bit types: mma.sync -----------------------------------------------------------------------------------------------------

// Up to 64 query rows: HBM bounds these, so the tiles stream through a ring of cp.async stages and the products only have to keep up.  A
// warp owns 16 keys of every tile and RM x 16 rows with a softmax of its own (reference, mass and sums in registers); the four warps that
// share rows are joined when the unit ends.  With the rows a block holds, WR = 1 or 2 rows of warps.
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
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

struct RowPtr { const char* k; const char* v; };

template <int DK, int DV, int WR> struct MmaShape {
    static constexpr int threads = WR * 128, stage = kTile * (DK + DV) * 2;
    static constexpr int stages = WR == 1 ? (stage > 24576 ? 3 : stage > 16384 ? 4 : 5) : (stage > 24576 ? 4 : 6);
    static constexpr int ring = 8;                             // of row pointers and key masks: at least stages + 2
    static_assert(stages + 2 <= ring, "");
    static constexpr int chunk = 32 + 4;                       // columns of a joining round, padded
};

template <typename T, int DK, int DV, int WR, int RM>
struct MmaSmem {
    using S = MmaShape<DK, DV, WR>;
    static constexpr int rows = WR * RM * 16;
    static constexpr int tiles = 0, ptrs = S::stages * S::stage, there = ptrs + S::ring * kTile * (int)sizeof(RowPtr), bad = there + S::ring * 8,
                         wm = bad + S::ring * 8, wl = wm + 4 * rows * 4, join = wl + 4 * rows * 4, total = join + 4 * rows * S::chunk * 4;
};

template <typename T, int DK, int DV, int WR, int RM>
__global__ void __launch_bounds__(WR * 128, WR == 1 ? 2 : 1) draft_mma_kernel(const __grid_constant__ DraftParams p) {
    using S = MmaShape<DK, DV, WR>;
    using L = MmaSmem<T, DK, DV, WR, RM>;
    constexpr int NT = S::threads, ST = S::stages, RING = S::ring, ROWS = L::rows, KP = DK / 8, VP = DV / 8;
    extern __shared__ __align__(128) unsigned char sm[];
    RowPtr* ptrs = reinterpret_cast<RowPtr*>(sm + L::ptrs);
    uint32_t* there = reinterpret_cast<uint32_t*>(sm + L::there);       // [ring][2]
    uint32_t* badw = reinterpret_cast<uint32_t*>(sm + L::bad);
    float* wm = reinterpret_cast<float*>(sm + L::wm);
    float* wl = reinterpret_cast<float*>(sm + L::wl);
    float* joinb = reinterpret_cast<float*>(sm + L::join);
    chain_enter();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, wk = w & 3, wr = w >> 2, kw = wk * 16, g = lane >> 2, r4 = lane & 3;
    Place at;
    int64_t x0 = 0, x1 = 0;
    const int64_t all = find_place<NT>(p, [&](int64_t n) {
        const int64_t parts = parts_of(p, n);
        x0 = part_start(blockIdx.x < parts ? blockIdx.x : 0, n, parts);
        x1 = part_start(blockIdx.x < parts ? blockIdx.x + 1 : 1, n, parts);
        return x0;
    }, at);
    if (blockIdx.x >= parts_of(p, all)) return;
    const int n_tiles = (int)(x1 - x0);
    bool bad = false;
    { bool b = false; draft_length(p, at.b, &b); bad |= b; }
    if (tid < 2 * RING) badw[tid] = 0;

    Place ahead = at;                  // of the tile whose row pointers are made next
    int made = 0;
    auto make_row = [&](const Place& pl, int tile, int j) {
        RowPtr rp{p.q, p.q};           // (never read: copies of rows that are not there have no source)
        const bool on = key_row(p, pl, pl.unit / p.row_tiles, j, rp.k, rp.v, &bad);
        const uint32_t m = __ballot_sync(0xffffffffu, on);
        if (lane == 0) there[(tile % RING) * 2 + (j >> 5)] = m;
        if (!on) rp = RowPtr{nullptr, nullptr};
        ptrs[(tile % RING) * kTile + j] = rp;
    };
    // the first stages' pointers at once: threads 0-63 the first tile, 64-127 the second, ...
    for (int i = 0; i < ST && i < n_tiles; ++i) {
        if ((i * 2) % (NT / 32) <= w && w < (i * 2) % (NT / 32) + 2) make_row(ahead, i, tid % 64);
        ahead.next(p);
        ++made;
    }
    __syncthreads();
    const uint32_t tiles_u = smem_u32(sm);
    auto issue = [&](int tile) {
        const uint32_t base = tiles_u + (tile % ST) * S::stage;
        const RowPtr* rows = ptrs + (tile % RING) * kTile;
#pragma unroll
        for (int i = 0; i < kTile * KP / NT; ++i) {
            const int x = i * NT + tid, j = x / KP, c = x % KP;
            const char* src = rows[j].k;
            const bool on = src != nullptr && c * 8 < p.K;
            cp_async16(base + j * (DK * 2) + ((c ^ (j & 7)) << 4), on ? src + c * 16 : p.q, on);
        }
#pragma unroll
        for (int i = 0; i < kTile * VP / NT; ++i) {
            const int x = i * NT + tid, j = x / VP, c = x % VP;
            const char* src = rows[j].v;
            const bool on = src != nullptr && c * 8 < p.V;
            cp_async16(base + kTile * DK * 2 + j * (DV * 2) + ((c ^ (j & 7)) << 4), on ? src + c * 16 : p.q, on);
        }
    };
    for (int i = 0; i < ST - 1; ++i) {
        if (i < n_tiles) issue(i);
        cp_async_commit();
    }

    uint32_t qf[RM][DK / 16][4];
    float o[RM][DV / 8][4], ref[RM][2], mass[RM][2];
    int first_tile = at.tile;
    bool fresh = true, first_piece = true;
    const uint32_t flip = p.neg ? 0x80008000u : 0u;
    for (int it = 0; it < n_tiles; ++it) {
        const bool draft = at.tile >= at.tiles - p.draft_tiles;
        if (fresh) {
            first_tile = at.tile;
            fresh = false;
#pragma unroll
            for (int m = 0; m < RM; ++m) {
                ref[m][0] = ref[m][1] = -INFINITY;
                mass[m][0] = mass[m][1] = 0.f;
#pragma unroll
                for (int d = 0; d < DV / 8; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[m][d][e] = 0.f;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    int n, h;
                    const bool on = row_of(p, at.unit, (wr * RM + m) * 16 + half * 8 + g, n, h);
                    const char* src = p.q + at.b * p.q_b + n * p.q_n + h * p.q_h + 4 * r4;
#pragma unroll
                    for (int ks = 0; ks < DK / 16; ++ks)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            qf[m][ks][half + 2 * e] = on && ks * 16 + e * 8 < p.K ? __ldg(reinterpret_cast<const uint32_t*>(src + ks * 32 + e * 16)) ^ flip : 0u;
                }
            }
        }
        cp_async_wait<ST - 2>();
        if (draft) {                   // what this thread has copied of the tile's values
            const uint32_t base = tiles_u + (it % ST) * S::stage + kTile * DK * 2;
#pragma unroll
            for (int i = 0; i < kTile * VP / NT; ++i) {
                const int x = i * NT + tid, j = x / VP, c = x % VP;
                if (take_out<T>(base + j * (DV * 2) + ((c ^ (j & 7)) << 4))) atomicOr(&badw[(it % RING) * 2 + (j >> 5)], 1u << (j & 31));
            }
        }
        __syncthreads();               // the tile is there, and so are the pointers made one round ago; its predecessor's stage is free
        if (it + ST - 1 < n_tiles) issue(it + ST - 1);
        cp_async_commit();
        if (made < n_tiles && made <= it + ST) {
            if (w < 2) make_row(ahead, made, tid);
            ahead.next(p);
            ++made;
        }
        if (tid < 2) badw[((it + 4) % RING) * 2 + tid] = 0;

        const uint32_t kbase = tiles_u + (it % ST) * S::stage, vbase = kbase + kTile * DK * 2;
        float s[RM][2][4];
#pragma unroll
        for (int m = 0; m < RM; ++m)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[m][nt][e] = 0.f;
        {
            const int row = kw + ((lane >> 4) << 3) + (lane & 7), c0 = (lane >> 3) & 1;
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
                uint32_t b[4];
                ldmatrix4(b, kbase + row * (DK * 2) + (((ks * 2 + c0) ^ (row & 7)) << 4));
#pragma unroll
                for (int m = 0; m < RM; ++m) {
                    Frag<T>::mma(s[m][0], qf[m][ks][0], qf[m][ks][1], qf[m][ks][2], qf[m][ks][3], b[0], b[1]);
                    Frag<T>::mma(s[m][1], qf[m][ks][0], qf[m][ks][1], qf[m][ks][2], qf[m][ks][3], b[2], b[3]);
                }
            }
        }
        const uint32_t keys = there[(it % RING) * 2 + (wk >> 1)] >> ((wk & 1) * 16) & 0xffffu;
        const uint32_t spoilt = draft ? badw[(it % RING) * 2 + (wk >> 1)] >> ((wk & 1) * 16) & 0xffffu : 0u;
        uint32_t seen[RM][2];
#pragma unroll
        for (int m = 0; m < RM; ++m) seen[m][0] = seen[m][1] = keys;
        if (draft) {
#pragma unroll
            for (int m = 0; m < RM; ++m) {
                int n, h;
                uint32_t mine = 0;
                const int tile0 = (at.tile - (at.tiles - p.draft_tiles)) * kTile;
                if (lane < 16 && row_of(p, at.unit, (wr * RM + m) * 16 + lane, n, h)) mine = (uint32_t)(draft_mask(p, at.b, n, tile0, &bad) >> kw) & 0xffffu;
                seen[m][0] &= __shfl_sync(0xffffffffu, mine, g);
                seen[m][1] &= __shfl_sync(0xffffffffu, mine, g + 8);
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
                    float t = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                    const float now = fmaxf(ref[m][half], t - kBias<T>);
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
            const int row = kw + (((lane >> 3) & 1) << 3) + (lane & 7), c0 = lane >> 4;
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
                uint32_t b[4];
                ldmatrix4_trans(b, vbase + row * (DV * 2) + (((d * 2 + c0) ^ (row & 7)) << 4));
#pragma unroll
                for (int m = 0; m < RM; ++m) {
                    Frag<T>::mma(o[m][2 * d], pf[m][0], pf[m][1], pf[m][2], pf[m][3], b[0], b[1]);
                    Frag<T>::mma(o[m][2 * d + 1], pf[m][0], pf[m][1], pf[m][2], pf[m][3], b[2], b[3]);
                }
            }
        }
        if (spoilt)
            for (int j = 0; j < 16; ++j) {
                if (!(spoilt >> j & 1)) continue;
                const int n = (at.tile - (at.tiles - p.draft_tiles)) * kTile + kw + j;
                const char* v = p.v + at.b * p.v_b + n * p.v_n + at.unit / p.row_tiles * p.v_h;
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
        const bool done = at.tile + 1 == at.tiles;
        if (done || it + 1 == n_tiles) {
            // the four warps of a row: one reference, sums added, 32 columns at a time
#pragma unroll
            for (int m = 0; m < RM; ++m)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float x = mass[m][half];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    const int row = (wr * RM + m) * 16 + half * 8 + g;
                    if (r4 == 0) { wm[wk * ROWS + row] = ref[m][half]; wl[wk * ROWS + row] = x; }
                }
            __syncthreads();
            const bool whole = done && first_tile == 0;
            float* slot = p.part + (int64_t)(2 * blockIdx.x + (first_piece ? 0 : 1)) * ROWS * (p.V + 2);
            float f[RM][2];
#pragma unroll
            for (int m = 0; m < RM; ++m)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = (wr * RM + m) * 16 + half * 8 + g;
                    const float t = fmaxf(fmaxf(wm[row], wm[ROWS + row]), fmaxf(wm[2 * ROWS + row], wm[3 * ROWS + row]));
                    f[m][half] = t == -INFINITY ? 1.f : ex2_approx(ref[m][half] - t);
                }
#pragma unroll
            for (int c = 0; c < DV / 32; ++c) {
#pragma unroll
                for (int m = 0; m < RM; ++m)
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int row = (wr * RM + m) * 16 + half * 8 + g;
                            *reinterpret_cast<float2*>(joinb + (wk * ROWS + row) * S::chunk + d * 8 + 2 * r4) =
                                make_float2(o[m][c * 4 + d][2 * half] * f[m][half], o[m][c * 4 + d][2 * half + 1] * f[m][half]);
                        }
                __syncthreads();
                for (int x = tid; x < ROWS * 8; x += NT) {
                    const int row = x >> 3, q = (x & 7) * 4, col = c * 32 + q;
                    int n, h;
                    if (!row_of(p, at.unit, row, n, h) || col >= p.V) continue;
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 y = *reinterpret_cast<const float4*>(joinb + (i * ROWS + row) * S::chunk + q);
                        sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
                    }
                    float t = -INFINITY, all_mass = 0.f;
                    if (whole || c == 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) t = fmaxf(t, wm[i * ROWS + row]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) all_mass += t == -INFINITY ? wl[i * ROWS + row] : wl[i * ROWS + row] * ex2_approx(wm[i * ROWS + row] - t);
                    }
                    if (whole) {
                        const bool real = is_draft(p, at.b, n);
                        const float inv = real ? finish_scale(all_mass) : 0.f;
                        const int64_t at_out = ((int64_t)at.b * p.N + n) * p.H + h;
                        uint2 y = make_uint2(Frag<T>::pack(sum.x * inv, sum.y * inv), Frag<T>::pack(sum.z * inv, sum.w * inv));
                        if (!real) y = make_uint2(0u, 0u);
                        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + at_out * p.V + col) = y;
                        if (p.lse && c == 0 && q == 0) p.lse[at_out] = real ? finish_lse(t, all_mass) : -INFINITY;
                    } else {
                        *reinterpret_cast<float4*>(slot + row * p.V + col) = sum;
                        if (c == 0 && q == 0) *reinterpret_cast<float2*>(slot + ROWS * p.V + 2 * row) = make_float2(t, all_mass);
                    }
                }
                __syncthreads();
            }
            first_piece = false;
            fresh = true;
        }
        const int b = at.b;
        at.next(p);
        if (at.b != b) { bool d = false; draft_length(p, at.b, &d); bad |= d; }
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
}

// ---- joining the parts -------------------------------------------------------------------------------------------------------

// Block (c, r) joins row r of the unit in which part c starts, if it is the first part that does.
constexpr int kJoinThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) draft_join_kernel(const __grid_constant__ DraftParams p) {
    __shared__ float red[kJoinThreads / 32][256];
    __shared__ float wm[kJoinThreads / 32], wl[kJoinThreads / 32];
    chain_enter();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, r = blockIdx.y;
    const int64_t c0 = blockIdx.x + 1;
    Place at;
    int64_t parts = 0, x0 = 0;
    const int64_t all = find_place<kJoinThreads>(p, [&](int64_t n) {
        parts = parts_of(p, n);
        x0 = c0 < parts ? part_start(c0, n, parts) : 0;
        return x0;
    }, at);
    if (c0 >= parts || at.tile == 0) return;                                 // (a part that starts with a unit)
    const int64_t u0 = x0 - at.tile, u1 = u0 + at.tiles;
    if (part_start(c0 - 1, all, parts) > u0) return;
    int n, h;
    if (!row_of(p, at.unit, r, n, h)) return;
    // parts c0 - 1 .. last touch the unit; the first of them in its last slot, unless the unit is all that it has
    int64_t last = c0;
    while (last + 1 < parts && part_start(last + 1, all, parts) < u1) ++last;
    const int64_t slots = last - c0 + 2, size = (int64_t)p.rows * (p.V + 2);
    auto slot_of = [&](int64_t i) {
        const int64_t c = c0 - 1 + i;
        return p.part + (2 * c + (i == 0 && part_start(c, all, parts) < u0 ? 1 : 0)) * size;
    };
    float top = -INFINITY;
    for (int64_t i = tid; i < slots; i += kJoinThreads) top = fmaxf(top, slot_of(i)[p.rows * p.V + 2 * r]);
    top = warp_max(top);
    if (lane == 0) wm[w] = top;
    __syncthreads();
    top = wm[0];
#pragma unroll
    for (int i = 1; i < kJoinThreads / 32; ++i) top = fmaxf(top, wm[i]);
    const float ref = top == -INFINITY ? 0.f : top;
    float mass = 0.f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};                       // columns lane*4 and lane*4 + 128
    for (int64_t i = w; i < slots; i += kJoinThreads / 32) {
        const float* s = slot_of(i);
        const float f = exp2f(s[p.rows * p.V + 2 * r] - ref);
        mass = fmaf(f, s[p.rows * p.V + 2 * r + 1], mass);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int col = half * 128 + lane * 4;
            if (col < p.V) {
                const float4 x = *reinterpret_cast<const float4*>(s + r * p.V + col);
                o[4 * half] = fmaf(f, x.x, o[4 * half]);
                o[4 * half + 1] = fmaf(f, x.y, o[4 * half + 1]);
                o[4 * half + 2] = fmaf(f, x.z, o[4 * half + 2]);
                o[4 * half + 3] = fmaf(f, x.w, o[4 * half + 3]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) red[w][(i >> 2) * 128 + lane * 4 + (i & 3)] = o[i];
    if (lane == 0) wl[w] = mass;
    __syncthreads();
    mass = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) mass += wl[i];
    const bool real = is_draft(p, at.b, n);
    const float inv = finish_scale(mass);
    const int64_t row = ((int64_t)at.b * p.N + n) * p.H + h;
    if (tid < p.V) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < kJoinThreads / 32; ++i) x += red[i][tid];
        reinterpret_cast<T*>(p.out)[row * p.V + tid] = from_f<T>(real ? x * inv : 0.f);
    }
    if (p.lse && tid == 0) p.lse[row] = real ? finish_lse(top, mass) : -INFINITY;
}

// ---- launches ----------------------------------------------------------------------------------------------------------------

static size_t generic_smem(const DraftParams& p) {
    const int VS = p.V > 128 ? 256 : 128;
    return ((size_t)kTile * (p.K + 4) + (size_t)kTile * VS + (size_t)kGenRows * p.K + (size_t)kGenRows * kTile) * 4;
}

static void fit_rows(DraftParams& p, int rows, int blocks) {
    p.rows = rows;
    p.row_tiles = (p.N * p.G + rows - 1) / rows;
    p.grid = blocks;
}

// Which kernel: 16-bit rows of up to 128 go to the tensor cores, with as many rows to a block as there are (16, 32 or 64).
enum { kGeneric = 0, kMma16, kMma32, kMma64 };
static void choose(DraftParams& p, int dtype) {
    const int sms = sm_count() > 0 ? sm_count() : 148, rows = p.N * p.G;
    if (dtype == HTREE_F32 || p.K > 128 || p.V > 128) {
        p.variant = kGeneric;
        fit_rows(p, kGenRows, sms * (generic_smem(p) <= 110 * 1024 ? 2 : 1));
        return;
    }
    p.variant = rows <= 16 ? kMma16 : rows <= 32 ? kMma32 : kMma64;
    fit_rows(p, rows <= 16 ? 16 : rows <= 32 ? 32 : 64, rows <= 16 ? 2 * sms : sms);
    if (p.c < 0.f) { p.neg = 1; p.c = -p.c; }
    if (p.c < 1.1754944e-38f) p.c = 1.1754944e-38f;        // a scale of zero: scores of zero, but what is masked stays minus infinity
}

template <typename T, int DK, int DV, int WR, int RM>
static int launch_mma(const DraftParams& p, cudaStream_t st) {
    static SmemLimit limit;
    constexpr size_t smem = MmaSmem<T, DK, DV, WR, RM>::total;
    if (const cudaError_t e = limit.raise((const void*)draft_mma_kernel<T, DK, DV, WR, RM>, smem)) return (int)e;
    return launch_chained(draft_mma_kernel<T, DK, DV, WR, RM>, dim3(p.grid), dim3(WR * 128), smem, st, p);
}
template <typename T, int DK, int DV>
static int launch_mma(const DraftParams& p, cudaStream_t st) {
    return p.variant == kMma16 ? launch_mma<T, DK, DV, 1, 1>(p, st) : p.variant == kMma32 ? launch_mma<T, DK, DV, 2, 1>(p, st) : launch_mma<T, DK, DV, 2, 2>(p, st);
}

template <typename T>
static int launch_generic(const DraftParams& p, cudaStream_t st) {
    static SmemLimit limit1, limit2;
    const size_t smem = generic_smem(p);
    if (p.V <= 128) {
        if (const cudaError_t e = limit1.raise((const void*)draft_generic_kernel<T, 1>, smem)) return (int)e;
        return launch_chained(draft_generic_kernel<T, 1>, dim3(p.grid), dim3(kGenThreads), smem, st, p);
    }
    if (const cudaError_t e = limit2.raise((const void*)draft_generic_kernel<T, 2>, smem)) return (int)e;
    return launch_chained(draft_generic_kernel<T, 2>, dim3(p.grid), dim3(kGenThreads), smem, st, p);
}

template <typename T>
static int launch_draft(const DraftParams& p, cudaStream_t st) {
    int rc;
    if constexpr (sizeof(T) == 4) {
        rc = launch_generic<T>(p, st);
    } else {
        rc = p.variant == kGeneric ? launch_generic<T>(p, st)
           : p.K <= 64 ? (p.V <= 64 ? launch_mma<T, 64, 64>(p, st) : launch_mma<T, 64, 128>(p, st))
                       : (p.V <= 64 ? launch_mma<T, 128, 64>(p, st) : launch_mma<T, 128, 128>(p, st));
    }
    if (rc || p.grid == 1) return rc;
    return launch_chained(draft_join_kernel<T>, dim3(p.grid - 1, p.rows), dim3(kJoinThreads), 0, st, p);
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
    p.B = d->B; p.N = d->N; p.H = d->H; p.Hkv = c->H_kv; p.G = d->H / c->H_kv; p.K = c->K; p.V = c->V; p.M = d->M; p.pages = c->pages;
    p.draft_tiles = (d->N + kTile - 1) / kTile;
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
    return (int64_t)p.grid * 2 * p.rows * (p.V + 2) * 4;
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
    if (workspace_bytes < (int64_t)p.grid * 2 * p.rows * (p.V + 2) * 4) return HTREE_E_SCRATCH;
    p.part = (float*)workspace;
    p.status = status;
    const cudaStream_t st = (cudaStream_t)stream;
    return cache->dtype == HTREE_F32 ? launch_draft<float>(p, st)
         : cache->dtype == HTREE_BF16 ? launch_draft<__nv_bfloat16>(p, st) : launch_draft<__half>(p, st);
}

}  // extern "C"
