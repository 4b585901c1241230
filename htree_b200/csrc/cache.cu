// The paged key/value cache: block tables and slot maps from request lengths, rows into their slots, pages as contiguous tensors.
// Each moves bytes and computes nothing: HBM bounds the large calls, the launch the small ones.
#include "cache.cuh"

namespace htree {

int sm_count() {
    static std::atomic<int> have[64] = {};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return 0; }
    if (dev < 64 && (n = have[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { cudaGetLastError(); return 0; }
    if (dev < 64) have[dev].store(n, std::memory_order_relaxed);
    return n;
}

// ---- plan -------------------------------------------------------------------------------------------------------------------

struct PlanParams {
    int32_t* lengths;
    const int32_t* counts;
    int32_t* table;
    int32_t* pool;
    int32_t* top;
    int64_t* slots;
    int32_t* taken;
    int32_t* status;
    int64_t table_stride;
    int32_t B, M, n, pool_size, slots_here;
    FastDiv page;
};

constexpr int kPlanThreads = 512;

// Exclusive scan over the block of one 64-bit value a thread; *total is the block's sum.  Two barriers.
__device__ __forceinline__ int64_t block_scan_i64(int64_t x, int64_t* scratch, int64_t* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int64_t in = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += y;
    }
    if (lane == 31) scratch[w] = in;
    __syncthreads();
    int64_t before = 0, tot = 0;
    for (int i = 0; i < kPlanThreads / 32; ++i) {
        const int64_t c = scratch[i];
        if (i < w) before += c;
        tot += c;
    }
    __syncthreads();
    *total = tot;
    return before + in - x;
}

// A request's length, clamped to what its table row can name (and so that a length rounded up to whole pages stays below 2^31).
__device__ __forceinline__ int plan_length(const PlanParams& p, int b, bool* bad) {
    int64_t room = (int64_t)p.M * p.page.d;
    if (room > 0x7fffffff - (int64_t)p.page.d) room = 0x7fffffff - (int64_t)p.page.d;
    int64_t len = p.lengths[b];
    if (len < 0 || len > room) { *bad = true; len = len < 0 ? 0 : room; }
    return (int)len;
}

// One cluster does the whole plan, so that the pages that ending rows give back can go to growing rows in the same call: every block
// computes the two scans for itself (a few words a request), the blocks share the rows, and cluster barriers separate the pushes, the
// pops and the slots.  `W` threads work on a row: a warp where there are many rows, all of them where there is one.
__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(const __grid_constant__ PlanParams p) {
    __shared__ int64_t scratch[kPlanThreads / 32];
    __shared__ int64_t first[kPlanThreads];
    __shared__ int32_t some[kPlanThreads], held[kPlanThreads], count[kPlanThreads];
    chain_enter();
    const int rank = (int)cluster_rank(), blocks = (int)cluster_blocks(), tid = threadIdx.x;
    const int me = rank * kPlanThreads + tid, all = blocks * kPlanThreads;
    bool bad = false, refused = false;
    int64_t top = *p.top;
    if (top < 0 || top > p.pool_size) { bad = true; top = top < 0 ? 0 : p.pool_size; }
    const int chunk_rows = p.B < kPlanThreads ? p.B : kPlanThreads;
    int W = 32;
    while (W * 2 * chunk_rows <= all) W *= 2;
    const int groups = all / W, group = me / W, lane = me % W;

    // rows that end: their pages onto the pool
    int64_t freed_all = 0;
    for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int64_t f = 0;
        if (b < p.B && p.counts[b] < 0) f = p.page.div((uint32_t)(plan_length(p, b, &bad) + (int64_t)p.page.d - 1));
        int64_t sum;
        const int64_t at = block_scan_i64(f, scratch, &sum);
        first[tid] = top + freed_all + at;
        some[tid] = (int32_t)f;
        __syncthreads();
        if (sum > 0)
            for (int r = group; r < kPlanThreads; r += groups)
                for (int j = lane; j < some[r]; j += W) {
                    int32_t* e = p.table + (int64_t)(b0 + r) * p.table_stride + j;
                    const int64_t to = first[r] + j;
                    if (to < p.pool_size) p.pool[to] = *e; else bad = true;       // more pages than the pool has: a table with repeats
                    *e = -1;
                }
        freed_all += sum;
        __syncthreads();
    }
    int64_t have = top + freed_all;
    if (have > p.pool_size) have = p.pool_size;
    cluster_sync();

    // rows that grow: pages from the pool's end
    int64_t need_all = 0, given_all = 0;
    for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int64_t need = 0;
        int c = 0, len = 0, h = 0;
        bool grows = false;
        if (b < p.B) {
            c = p.counts[b];
            if (c > 0) {
                len = plan_length(p, b, &bad);
                h = (int)p.page.div((uint32_t)(len + (int64_t)p.page.d - 1));
                const int64_t now = (int64_t)len + c;
                grows = c <= p.n && now <= (int64_t)p.M * p.page.d && now < (int64_t(1) << 31) - p.page.d;
                if (!grows) refused = true;
                else need = p.page.div((uint32_t)(now + (int64_t)p.page.d - 1)) - h;
            }
        }
        int64_t sum, dummy;
        const int64_t at = need_all + block_scan_i64(need, scratch, &sum);
        const bool served = grows && (need == 0 || at + need <= have);
        (void)block_scan_i64(served ? need : 0, scratch, &dummy);
        given_all += dummy;
        need_all += sum;
        first[tid] = have - 1 - at;
        some[tid] = served ? (int32_t)need : 0;
        held[tid] = h;
        count[tid] = served ? c : 0;
        __syncthreads();
        for (int r = group; r < kPlanThreads; r += groups)
            for (int j = lane; j < some[r]; j += W)
                p.table[(int64_t)(b0 + r) * p.table_stride + held[r] + j] = p.pool[first[r] - j];
        if (rank == 0 && b < p.B) p.taken[b] = count[tid];
        __syncthreads();
    }
    cluster_sync();          // nobody reads lengths, counts or top any more, and the tables are complete
    if (p.slots_here)
        for (int b0 = 0; b0 < p.B; b0 += groups) {
            const int b = b0 + group;
            if (b >= p.B) continue;
            const int c = p.taken[b];
            bool dull = false;
            const int len = c > 0 ? plan_length(p, b, &dull) : 0;
            for (int i = lane; i < p.n; i += W) {
                int64_t s = -1;
                if (i < c) {
                    const uint32_t pos = (uint32_t)(len + i), pg = p.page.div(pos);
                    s = (int64_t)p.table[(int64_t)b * p.table_stride + pg] * p.page.d + (pos - pg * p.page.d);
                }
                p.slots[(int64_t)b * p.n + i] = s;
            }
        }
    cluster_sync();          // ... nor here
    for (int b = me; b < p.B; b += all) {
        bool dull = false;
        if (p.counts[b] < 0) p.lengths[b] = 0;
        else if (p.taken[b] > 0) p.lengths[b] = plan_length(p, b, &dull) + p.taken[b];
    }
    if (me == 0) *p.top = (int32_t)(have - given_all);
    if (p.status) {
        if (bad) atomicOr(p.status, HTREE_STATUS_CACHE);
        if (refused) atomicOr(p.status, HTREE_STATUS_ROW);
    }
}

// The slot map of a plan with many new tokens, by the whole chip (8 bytes a token; the cluster alone would write it at a tenth of the
// rate).  Lengths have been advanced already.
constexpr int kSlotsPerThread = 4;
__global__ void __launch_bounds__(256) cache_slots_kernel(const __grid_constant__ PlanParams p) {
    chain_enter();
    const int b = blockIdx.y, c = p.taken[b];
    const int64_t start = (int64_t)p.lengths[b] - c;
    const int32_t* row = p.table + (int64_t)b * p.table_stride;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x); i < p.n; i += (int64_t)gridDim.x * 256) {
        int64_t s = -1;
        if (i < c) {
            const uint32_t pos = (uint32_t)(start + i), pg = p.page.div(pos);
            s = (int64_t)row[pg] * p.page.d + (pos - pg * p.page.d);
        }
        p.slots[(int64_t)b * p.n + i] = s;
    }
}

// ---- append and gather ------------------------------------------------------------------------------------------------------

// A token's row over all heads, keys first, as 16-byte pieces; a thread keeps its piece and goes from token to token.
struct MoveParams {
    char* ck;
    char* cv;
    const char* k;
    const char* v;
    char* ok;
    char* ov;
    const int64_t* slots;
    const int32_t* index;
    const int32_t* table;
    const int32_t* lengths;
    int32_t* status;
    int64_t ck_page, ck_row, ck_head, cv_page, cv_row, cv_head;      // all strides in bytes
    int64_t k_b, k_n, k_head, v_b, v_n, v_head;
    int64_t table_stride, tokens, slots_all;
    int32_t N, n, pages, M, pk, pv, H_kv, px;                         // pk, pv: pieces of a head's key and value row
    FastDiv page, per_row;
};

struct Piece {
    bool on, key;
    int head, at;       // byte within the head's row
};
__device__ __forceinline__ Piece piece_of(const MoveParams& p) {
    Piece x;
    const int i = blockIdx.y * p.px + threadIdx.x % p.px, keys = p.H_kv * p.pk;
    x.on = i < p.H_kv * (p.pk + p.pv) && (int)threadIdx.x < p.px * (int)(blockDim.x / p.px);
    x.key = i < keys;
    const int j = x.key ? i : i - keys, per = x.key ? p.pk : p.pv;
    x.head = j / per;
    x.at = (j - x.head * per) * 16;
    return x;
}

constexpr int kMoveUnroll = 4;

__global__ void __launch_bounds__(256) cache_append_kernel(const __grid_constant__ MoveParams p) {
    chain_enter();
    const Piece x = piece_of(p);
    if (!x.on) return;
    const int py = blockDim.x / p.px;
    const int64_t step = (int64_t)gridDim.x * py;
    char* dst0 = x.key ? p.ck + x.head * p.ck_head + x.at : p.cv + x.head * p.cv_head + x.at;
    const char* src0 = x.key ? p.k + x.head * p.k_head + x.at : p.v + x.head * p.v_head + x.at;
    const int64_t d_page = x.key ? p.ck_page : p.cv_page, d_row = x.key ? p.ck_row : p.cv_row;
    const int64_t s_b = x.key ? p.k_b : p.v_b, s_n = x.key ? p.k_n : p.v_n;
    bool bad = false;
    for (int64_t t0 = (int64_t)blockIdx.x * py + threadIdx.x / p.px; t0 < p.tokens; t0 += step * kMoveUnroll) {
        char* dst[kMoveUnroll];
        uint4 val[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const int64_t t = t0 + u * step;
            dst[u] = nullptr;
            if (t >= p.tokens) continue;
            const int64_t slot = p.slots[t];
            if (slot < 0 || slot >= p.slots_all) { bad |= slot != -1; continue; }
            const int b = (int)p.per_row.div((uint32_t)t), i = (int)(t - (int64_t)b * p.n);
            const int src = p.index ? p.index[t] : i;
            if (src < 0 || src >= p.N) { bad = true; continue; }
            const int64_t pg = slot / p.page.d;
            dst[u] = dst0 + pg * d_page + (slot - pg * p.page.d) * d_row;
            val[u] = __ldg(reinterpret_cast<const uint4*>(src0 + b * s_b + src * s_n));
        }
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            if (dst[u]) *reinterpret_cast<uint4*>(dst[u]) = val[u];
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
}

__global__ void __launch_bounds__(256) cache_gather_kernel(const __grid_constant__ MoveParams p) {
    chain_enter();
    const Piece x = piece_of(p);
    if (!x.on) return;
    const int py = blockDim.x / p.px;
    const int64_t step = (int64_t)gridDim.x * py;
    const char* src0 = x.key ? p.ck + x.head * p.ck_head + x.at : p.cv + x.head * p.cv_head + x.at;
    const int64_t s_page = x.key ? p.ck_page : p.cv_page, s_row = x.key ? p.ck_row : p.cv_row;
    const int64_t width = (int64_t)(x.key ? p.pk : p.pv) * 16;
    char* dst0 = (x.key ? p.ok : p.ov) + x.head * width + x.at;
    const int64_t d_row = p.H_kv * width;
    const int b = blockIdx.z;
    int64_t len = p.lengths[b];
    bool bad = len < 0 || len > (int64_t)p.M * p.page.d;
    if (bad) len = len < 0 ? 0 : (int64_t)p.M * p.page.d;
    const int32_t* row = p.table + (int64_t)b * p.table_stride;
    for (int64_t t0 = (int64_t)blockIdx.x * py + threadIdx.x / p.px; t0 < p.n; t0 += step * kMoveUnroll) {
        uint4 val[kMoveUnroll];
        int32_t pg[kMoveUnroll];
        uint32_t in[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const int64_t t = t0 + u * step;
            pg[u] = -1;
            if (t >= p.n || t >= len) continue;
            const uint32_t i = p.page.div((uint32_t)t);
            in[u] = (uint32_t)t - i * p.page.d;
            pg[u] = row[i];
            if (pg[u] < 0 || pg[u] >= p.pages) { bad = true; pg[u] = -1; }
        }
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            val[u] = pg[u] < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(src0 + pg[u] * s_page + in[u] * s_row));
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const int64_t t = t0 + u * step;
            if (t < p.n) *reinterpret_cast<uint4*>(dst0 + ((int64_t)b * p.n + t) * d_row) = val[u];
        }
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
}

static void fill_move(MoveParams& p, const HtreeCache& c, int32_t* status) {
    const int es = cache_esize(c.dtype);
    p = MoveParams{};
    p.ck = (char*)c.k; p.cv = (char*)c.v;
    p.ck_page = c.k_page * es; p.ck_row = c.k_row * es; p.ck_head = c.k_head * es;
    p.cv_page = c.v_page * es; p.cv_row = c.v_row * es; p.cv_head = c.v_head * es;
    p.pages = c.pages; p.H_kv = c.H_kv; p.pk = c.K * es / 16; p.pv = c.V * es / 16;
    p.page = FastDiv((uint32_t)c.page_size); p.slots_all = (int64_t)c.pages * c.page_size;
    p.status = status;
    const int pieces = c.H_kv * (p.pk + p.pv);
    p.px = pieces < 256 ? pieces : 256;
}

}  // namespace htree

using namespace htree;

extern "C" {

int htree_b200_cache_plan(int32_t B, int32_t M, int32_t page_size, int32_t n, int32_t* lengths, const int32_t* counts, int32_t* table,
                          int64_t table_stride, int32_t* pool, int32_t pool_size, int32_t* top, int64_t* slots, int32_t* taken,
                          int32_t* status, void* stream) {
    if (!lengths || !counts || !table || !pool || !top || !slots || !taken) return HTREE_E_NULL;
    if (B <= 0 || M <= 0 || page_size <= 0 || n <= 0 || pool_size <= 0 || table_stride < M) return HTREE_E_SHAPE;
    if (B > 65535 || page_size > (1 << 20)) return HTREE_E_UNSUPPORTED;
    PlanParams p{};
    p.lengths = lengths; p.counts = counts; p.table = table; p.pool = pool; p.top = top; p.slots = slots; p.taken = taken; p.status = status;
    p.table_stride = table_stride; p.B = B; p.M = M; p.n = n; p.pool_size = pool_size;
    p.page = FastDiv((uint32_t)page_size);
    const int64_t entries = (int64_t)B * M, map = (int64_t)B * n;
    p.slots_here = map <= 16384;
    const int CL = entries <= 4096 ? 1 : 8;
    const int rc = launch_clusters(cache_plan_kernel, CL, dim3(1), dim3(kPlanThreads), 0, (cudaStream_t)stream, p);
    if (rc || p.slots_here) return rc;
    int64_t gx = (n + 256 * kSlotsPerThread - 1) / (256 * kSlotsPerThread);
    if (gx > 4096) gx = 4096;
    return launch_chained(cache_slots_kernel, dim3((unsigned)gx, B), dim3(256), 0, (cudaStream_t)stream, p);
}

int htree_b200_cache_append(const HtreeCache* cache, int32_t B, int32_t N, int32_t n, const void* k, const int64_t* k_stride,
                            const void* v, const int64_t* v_stride, const int64_t* slots, const int32_t* index, int32_t* status,
                            void* stream) {
    if (const int rc = check_cache(cache)) return rc;
    if (!k || !v || !k_stride || !v_stride || !slots) return HTREE_E_NULL;
    if (B <= 0 || N <= 0 || n <= 0 || (!index && n > N)) return HTREE_E_SHAPE;
    if ((int64_t)B * n >= (int64_t(1) << 31)) return HTREE_E_UNSUPPORTED;
    const int es = cache_esize(cache->dtype);
    if (!cache_aligned(k) || !cache_aligned(v) || !cache_strides_ok(k_stride, es) || !cache_strides_ok(v_stride, es)) return HTREE_E_ALIGN;
    MoveParams p;
    fill_move(p, *cache, status);
    p.k = (const char*)k; p.v = (const char*)v; p.slots = slots; p.index = index;
    p.k_b = k_stride[0] * es; p.k_n = k_stride[1] * es; p.k_head = k_stride[2] * es;
    p.v_b = v_stride[0] * es; p.v_n = v_stride[1] * es; p.v_head = v_stride[2] * es;
    p.N = N; p.n = n; p.tokens = (int64_t)B * n; p.per_row = FastDiv((uint32_t)n);
    const int py = 256 / p.px, pieces = p.H_kv * (p.pk + p.pv), gy = (pieces + p.px - 1) / p.px;
    int64_t gx = (p.tokens + (int64_t)py * kMoveUnroll - 1) / ((int64_t)py * kMoveUnroll);
    if (gx > 1 << 20) gx = 1 << 20;
    return launch_chained(cache_append_kernel, dim3((unsigned)gx, gy), dim3(256), 0, (cudaStream_t)stream, p);
}

int htree_b200_cache_gather(const HtreeCache* cache, int32_t B, int32_t M, int32_t T, const int32_t* table, int64_t table_stride,
                            const int32_t* lengths, void* k, void* v, int32_t* status, void* stream) {
    if (const int rc = check_cache(cache)) return rc;
    if (!table || !lengths || !k || !v) return HTREE_E_NULL;
    if (B <= 0 || M <= 0 || T <= 0 || table_stride < M) return HTREE_E_SHAPE;
    if (B > 65535) return HTREE_E_UNSUPPORTED;
    if (!cache_aligned(k) || !cache_aligned(v)) return HTREE_E_ALIGN;
    MoveParams p;
    fill_move(p, *cache, status);
    p.ok = (char*)k; p.ov = (char*)v; p.table = table; p.table_stride = table_stride; p.lengths = lengths; p.M = M; p.n = T;
    const int py = 256 / p.px, pieces = p.H_kv * (p.pk + p.pv), gy = (pieces + p.px - 1) / p.px;
    int64_t gx = (T + (int64_t)py * kMoveUnroll - 1) / ((int64_t)py * kMoveUnroll);
    if (gx > 1 << 20) gx = 1 << 20;
    return launch_chained(cache_gather_kernel, dim3((unsigned)gx, gy, B), dim3(256), 0, (cudaStream_t)stream, p);
}

}  // extern "C"
