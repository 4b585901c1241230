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

static void choose(DraftParams& p, int dtype) {
    const int sms = sm_count() > 0 ? sm_count() : 148;
    const size_t smem = generic_smem(p);
    fit_rows(p, kGenRows, sms * (smem <= 110 * 1024 ? 2 : 1));
}

template <typename T>
static int launch_draft(const DraftParams& p, cudaStream_t st) {
    int rc;
    static SmemLimit limit1, limit2;
    const size_t smem = generic_smem(p);
    if (p.V <= 128) {
        if (const cudaError_t e = limit1.raise((const void*)draft_generic_kernel<T, 1>, smem)) return (int)e;
        rc = launch_chained(draft_generic_kernel<T, 1>, dim3(p.grid), dim3(kGenThreads), smem, st, p);
    } else {
        if (const cudaError_t e = limit2.raise((const void*)draft_generic_kernel<T, 2>, smem)) return (int)e;
        rc = launch_chained(draft_generic_kernel<T, 2>, dim3(p.grid), dim3(kGenThreads), smem, st, p);
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
