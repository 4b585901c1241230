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
    int32_t room;          // tokens that a row can name, and below 2^31 when rounded up to whole pages
    FastDiv page;
};

constexpr int kPlanThreads = 1024;
constexpr uint32_t kPlanMost = 0x7fffffffu;      // sums of pages stop here: no pool has as many

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kPlanMost); }

// Exclusive scan over the block of one count a thread, saturating; *total is the block's sum.  Two barriers.
__device__ __forceinline__ uint32_t block_scan_sat(uint32_t x, uint32_t* scratch, uint32_t* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint32_t in = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in = sat_add(in, y);
    }
    uint32_t before = __shfl_up_sync(0xffffffffu, in, 1);
    if (lane == 0) before = 0;
    if (lane == 31) scratch[w] = in;
    __syncthreads();
    uint32_t sum = lane < kPlanThreads / 32 ? scratch[lane] : 0;       // every warp scans the warps' sums
#pragma unroll
    for (int o = 1; o < kPlanThreads / 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum = sat_add(sum, y);
    }
    *total = __shfl_sync(0xffffffffu, sum, kPlanThreads / 32 - 1);
    const uint32_t warps = __shfl_sync(0xffffffffu, sum, w > 0 ? w - 1 : 0);
    __syncthreads();
    return w > 0 ? sat_add(before, warps) : before;
}

// A request's length, clamped to what its table row can name (and so that a length rounded up to whole pages stays below 2^31).
__device__ __forceinline__ int plan_length(const PlanParams& p, int len, bool* bad) {
    const int in = min(max(len, 0), p.room);
    if (in != len) *bad = true;
    return in;
}

// One cluster does the whole plan, so that the pages that ending rows give back can go to growing rows in the same call: every block
// computes the two scans for itself (a few words a request), the blocks share the rows, and cluster barriers separate the pushes, the
// pops and the slots.  `W` threads work on a row: a warp where there are many rows, all of them where there is one.  What bounds it is
// latency: entries move eight at a time (one by one, 512 rows of 800 pages took 61 us; so 12), by sixteen blocks of 1024 threads (admitting,
// extending and ending 512 requests of 16384 tokens in pages of 16: 40 us in three calls, by eight of 512 threads 50; 1024 requests of 2000 in
// pages of one: 56 and 108).
__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(const __grid_constant__ PlanParams p) {
    __shared__ uint32_t scratch[kPlanThreads / 32];
    __shared__ uint32_t first[kPlanThreads];
    __shared__ int32_t some[kPlanThreads], held[kPlanThreads], count[kPlanThreads], start[kPlanThreads];
    chain_enter();
    const int rank = (int)cluster_rank(), blocks = (int)cluster_blocks(), tid = threadIdx.x;
    const int me = rank * kPlanThreads + tid, all = blocks * kPlanThreads;
    bool bad = false, refused = false;
    uint32_t top = (uint32_t)max(*p.top, 0);
    int count0 = 0, length0 = 0;                     // of the first rows, which are all rows of most batches
    if (tid < p.B) { count0 = p.counts[tid]; length0 = p.lengths[tid]; }
    if (top > (uint32_t)p.pool_size || *p.top < 0) { bad = true; top = min(top, (uint32_t)p.pool_size); }
    const int chunk_rows = p.B < kPlanThreads ? p.B : kPlanThreads;
    int log_w = 5;
    while (((2 << log_w) * chunk_rows) <= all) ++log_w;
    const int W = 1 << log_w, groups = all >> log_w, group = me >> log_w, lane = me & (W - 1);

    // rows that end: their pages onto the pool
    uint32_t freed_all = 0;
    const bool ends = __syncthreads_or(count0 < 0) || p.B > kPlanThreads;
    if (ends) {
        for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
            const int b = b0 + tid;
            uint32_t f = 0;
            if (b < p.B && (b0 ? p.counts[b] : count0) < 0)
                f = p.page.div((uint32_t)plan_length(p, b0 ? p.lengths[b] : length0, &bad) + p.page.d - 1);
            uint32_t sum;
            const uint32_t at = block_scan_sat(f, scratch, &sum);
            first[tid] = sat_add(top, sat_add(freed_all, at));
            some[tid] = (int32_t)f;
            __syncthreads();
            if (sum > 0)
                for (int r = group; r < chunk_rows; r += groups) {
                    int32_t* row = p.table + (int64_t)(b0 + r) * p.table_stride;
                    for (int j0 = lane; j0 < some[r]; j0 += 8 * W) {
                        int32_t e[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) if (j0 + u * W < some[r]) e[u] = row[j0 + u * W];
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            if (j0 + u * W < some[r]) {
                                const uint32_t to = first[r] + (uint32_t)(j0 + u * W);
                                if (to < (uint32_t)p.pool_size) p.pool[to] = e[u]; else bad = true;       // more pages than the pool has: a table with repeats
                                bad |= e[u] < 0;                                                          // a length of more pages than the row has
                                row[j0 + u * W] = -1;
                            }
                    }
                }
            freed_all = sat_add(freed_all, sum);
            __syncthreads();
        }
        cluster_sync();
    }
    const uint32_t have = min(sat_add(top, freed_all), (uint32_t)p.pool_size);

    // rows that grow: pages from the pool's end
    uint32_t need_all = 0, given_all = 0;
    for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        uint32_t need = 0;
        int c = 0, len = 0, h = 0;
        bool grows = false;
        if (b < p.B) {
            c = b0 ? p.counts[b] : count0;
            if (c > 0) {
                len = plan_length(p, b0 ? p.lengths[b] : length0, &bad);
                h = (int)p.page.div((uint32_t)len + p.page.d - 1);
                grows = c <= p.n && c <= p.room - len;
                if (!grows) refused = true;
                else need = p.page.div((uint32_t)(len + c) + p.page.d - 1) - h;
            }
        }
        uint32_t sum, given;
        const uint32_t at = sat_add(need_all, block_scan_sat(need, scratch, &sum));
        const bool served = grows && (need == 0 || sat_add(at, need) <= have);
        (void)block_scan_sat(served ? need : 0, scratch, &given);
        given_all += given;
        need_all = sat_add(need_all, sum);
        first[tid] = have - 1 - at;
        some[tid] = served ? (int32_t)need : 0;
        held[tid] = h;
        count[tid] = served ? c : 0;
        start[tid] = len;
        if (rank == 0 && b < p.B) p.taken[b] = served ? c : 0;
        __syncthreads();
        for (int r = group; r < chunk_rows; r += groups) {
            int32_t* row = p.table + (int64_t)(b0 + r) * p.table_stride + held[r];
            for (int j0 = lane; j0 < some[r]; j0 += 8 * W) {
                int32_t e[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) if (j0 + u * W < some[r]) e[u] = p.pool[first[r] - (uint32_t)(j0 + u * W)];
#pragma unroll
                for (int u = 0; u < 8; ++u) if (j0 + u * W < some[r]) row[j0 + u * W] = e[u];           // (every one is asked for a slot: looked at there)
            }
        }
        if (p.slots_here) {
            // a row's entries are written by the threads of its group: those of a warp see one another's after a warp's barrier, those of
            // several after the block's or the cluster's
            if (W == 32) __syncwarp(); else if (W <= kPlanThreads && blocks == 1) __syncthreads(); else cluster_sync();
            for (int r = group; r < chunk_rows; r += groups) {
                if (b0 + r >= p.B) break;
                for (int i = lane; i < p.n; i += W) {
                    int64_t s = -1;
                    if (i < count[r]) {
                        const uint32_t pos = (uint32_t)(start[r] + i), pg = p.page.div(pos);
                        const int32_t e = p.table[(int64_t)(b0 + r) * p.table_stride + pg];
                        if (e >= 0) s = (int64_t)e * p.page.d + (pos - pg * p.page.d); else bad = true;
                    }
                    p.slots[(int64_t)(b0 + r) * p.n + i] = s;
                }
            }
        }
        __syncthreads();
        if (p.B <= kPlanThreads) {
            if (blocks > 1) cluster_sync();              // nobody reads lengths, counts or top any more
            if (rank == 0 && b < p.B && (c < 0 || count[tid] > 0)) p.lengths[b] = c < 0 ? 0 : len + count[tid];
        }
    }
    if (p.B > kPlanThreads) {
        cluster_sync();
        for (int b = me; b < p.B; b += all) {
            bool dull = false;
            if (p.counts[b] < 0) p.lengths[b] = 0;
            else if (p.taken[b] > 0) p.lengths[b] = plan_length(p, p.lengths[b], &dull) + p.taken[b];
        }
    }
    if (me == 0) *p.top = (int32_t)(have - given_all);
    if (p.status) {
        if (bad) atomicOr(p.status, HTREE_STATUS_CACHE);
        if (refused) atomicOr(p.status, HTREE_STATUS_ROW);
    }
}

// Clusters of sixteen blocks have to be allowed, once per device.
static bool sixteen_allowed() {
    static std::atomic<int> have[64] = {};           // 1: allowed, 2: refused
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return false; }
    if (dev < 64 && have[dev].load(std::memory_order_acquire)) return have[dev].load(std::memory_order_acquire) == 1;
    const bool ok = cudaFuncSetAttribute((const void*)cache_plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
    if (!ok) cudaGetLastError();
    if (dev < 64) have[dev].store(ok ? 1 : 2, std::memory_order_release);
    return ok;
}

// The slot map of a plan with many new tokens, by the whole chip (8 bytes a token; the cluster alone would write it at a tenth of the
// rate).  Lengths have been advanced already.
constexpr int kSlotsPerThread = 8;
template <bool Pairs>
__global__ void __launch_bounds__(256) cache_slots_kernel(const __grid_constant__ PlanParams p) {
    chain_enter();
    const int b = blockIdx.y, c = p.taken[b];
    const int64_t start = (int64_t)p.lengths[b] - c;
    const int32_t* row = p.table + (int64_t)b * p.table_stride;
    bool bad = false;
    auto slot = [&](int64_t i) -> int64_t {
        if (i >= c) return -1;
        const uint32_t pos = (uint32_t)(start + i), pg = p.page.div(pos);
        const int32_t e = row[pg];
        if (e < 0) { bad = true; return -1; }
        return (int64_t)e * p.page.d + (pos - pg * p.page.d);
    };
    constexpr int V = Pairs ? 2 : 1;                 // slots of a store: two where a row starts on 16 bytes
    int64_t* out = p.slots + (int64_t)b * p.n;
#pragma unroll
    for (int u = 0; u < kSlotsPerThread / V; ++u) {
        const int64_t i = ((int64_t)blockIdx.x * (kSlotsPerThread / V) + u) * 256 * V + threadIdx.x * V;
        if (i >= p.n) break;
        if (Pairs) *reinterpret_cast<longlong2*>(out + i) = make_longlong2(slot(i), slot(i + 1));
        else out[i] = slot(i);
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
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
    int32_t N, n, pages, room, pk, pv, H_kv, px;                      // pk, pv: pieces of a head's key and value row; room: tokens of a table row
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

// As many blocks as stay resident, each of which goes on to its next tokens: their slots or pages are read while the present ones move.
// Four tokens of a thread in flight, four blocks of an SM: 65536 tokens of 1 KB are appended in 23.6 us (87% of the copy
// rate) and 4 x 65536 gathered at 96%; with 2 x 8, 8 x 4 or 4 x 6 the append takes 29, 33 and 31 us, the gather up to 4/3 as long.
constexpr int kMoveUnroll = 4, kMoveBlocks = 4;

__global__ void __launch_bounds__(256, kMoveBlocks) cache_append_kernel(const __grid_constant__ MoveParams p) {
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
    int64_t next[kMoveUnroll];
    auto look = [&](int64_t t0) {
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) next[u] = t0 + u * step < p.tokens ? __ldg(p.slots + t0 + u * step) : -1;
    };
    int64_t t0 = (int64_t)blockIdx.x * py + threadIdx.x / p.px;
    look(t0);
    for (; t0 < p.tokens; t0 += step * kMoveUnroll) {
        char* dst[kMoveUnroll];
        uint4 val[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const int64_t t = t0 + u * step, slot = next[u];
            dst[u] = nullptr;
            if (slot < 0 || slot >= p.slots_all) { bad |= slot != -1; continue; }
            const uint32_t b = p.per_row.div((uint32_t)t), i = (uint32_t)t - b * (uint32_t)p.n;
            const int src = p.index ? __ldg(p.index + t) : (int)i;
            if (src < 0 || src >= p.N) { bad = true; continue; }
            // (slots below 2^31 go by the multiplication; a cache of more needs the division)
            const int64_t pg = slot >> 31 ? slot / p.page.d : p.page.div((uint32_t)slot);
            dst[u] = dst0 + pg * d_page + (slot - pg * p.page.d) * d_row;
            val[u] = __ldg(reinterpret_cast<const uint4*>(src0 + b * s_b + src * s_n));
        }
        look(t0 + step * kMoveUnroll);
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            if (dst[u]) *reinterpret_cast<uint4*>(dst[u]) = val[u];
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
}

__global__ void __launch_bounds__(256, kMoveBlocks) cache_gather_kernel(const __grid_constant__ MoveParams p) {
    chain_enter();
    const Piece x = piece_of(p);
    if (!x.on) return;
    const int py = blockDim.x / p.px;
    const int64_t step = (int64_t)gridDim.x * py;
    const char* src0 = x.key ? p.ck + x.head * p.ck_head + x.at : p.cv + x.head * p.cv_head + x.at;
    const int64_t s_page = x.key ? p.ck_page : p.cv_page, s_row = x.key ? p.ck_row : p.cv_row;
    const int64_t width = (int64_t)(x.key ? p.pk : p.pv) * 16, d_row = p.H_kv * width;
    char* dst0 = (x.key ? p.ok : p.ov) + x.head * width + x.at;
    bool bad = false;
    // tokens of all requests in one line, p.n of a request
    int32_t page[kMoveUnroll];
    uint32_t in[kMoveUnroll];
    auto look = [&](int64_t t0) {
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const int64_t t = t0 + u * step;
            page[u] = -1;
            if (t >= p.tokens) continue;
            const uint32_t b = p.per_row.div((uint32_t)t), pos = (uint32_t)t - b * (uint32_t)p.n;
            const int len = __ldg(p.lengths + b);
            if (len < 0 || len > p.room) bad = true;
            if ((int)pos >= min(len, p.room)) continue;
            const uint32_t i = p.page.div(pos);
            in[u] = pos - i * p.page.d;
            page[u] = __ldg(p.table + (int64_t)b * p.table_stride + i);
            if (page[u] < 0 || page[u] >= p.pages) { bad = true; page[u] = -1; }
        }
    };
    int64_t t0 = (int64_t)blockIdx.x * py + threadIdx.x / p.px;
    look(t0);
    for (; t0 < p.tokens; t0 += step * kMoveUnroll) {
        uint4 val[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            val[u] = page[u] < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(src0 + page[u] * s_page + in[u] * s_row));
        look(t0 + step * kMoveUnroll);
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const int64_t t = t0 + u * step;
            if (t < p.tokens) __stcs(reinterpret_cast<uint4*>(dst0 + t * d_row), val[u]);
        }
    }
    if (bad && p.status) atomicOr(p.status, HTREE_STATUS_CACHE);
}

// Blocks along the tokens: as many as there is work for, up to what is resident.
static dim3 move_grid(const MoveParams& p) {
    const int py = 256 / p.px, pieces = p.H_kv * (p.pk + p.pv), gy = (pieces + p.px - 1) / p.px, sms = sm_count() > 0 ? sm_count() : 148;
    const int64_t each = (int64_t)py * kMoveUnroll, want = (p.tokens + each - 1) / each;
    int64_t most = ((int64_t)sms * kMoveBlocks + gy - 1) / gy;
    // few tokens: a thread one token, so that all SMs help
    if (want < most) { const int64_t one = (p.tokens + py - 1) / py; return dim3((unsigned)(one < most ? one : most), gy); }
    return dim3((unsigned)most, gy);
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
    const int64_t entries = (int64_t)B * M, map = (int64_t)B * n, room = (int64_t)M * page_size, most = 0x7fffffff - (int64_t)page_size;
    p.room = (int32_t)(room < most ? room : most);
    p.slots_here = map <= 16384;
    const int CL = entries <= 4096 ? 1 : sixteen_allowed() ? 16 : 8;
    int rc = launch_chained_clusters(cache_plan_kernel, CL, dim3(CL), dim3(kPlanThreads), 0, (cudaStream_t)stream, p);
    if (rc && CL == 16) rc = launch_chained_clusters(cache_plan_kernel, 8, dim3(8), dim3(kPlanThreads), 0, (cudaStream_t)stream, p);
    if (rc && CL > 1) rc = launch_chained_clusters(cache_plan_kernel, 1, dim3(1), dim3(kPlanThreads), 0, (cudaStream_t)stream, p);
    if (rc || p.slots_here) return rc;
    const dim3 grid((unsigned)((n + 256 * (int64_t)kSlotsPerThread - 1) / (256 * kSlotsPerThread)), B);
    return n % 2 == 0 && cache_aligned(slots) ? launch_chained(cache_slots_kernel<true>, grid, dim3(256), 0, (cudaStream_t)stream, p)
                                              : launch_chained(cache_slots_kernel<false>, grid, dim3(256), 0, (cudaStream_t)stream, p);
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
    return launch_chained(cache_append_kernel, move_grid(p), dim3(256), 0, (cudaStream_t)stream, p);
}

int htree_b200_cache_gather(const HtreeCache* cache, int32_t B, int32_t M, int32_t T, const int32_t* table, int64_t table_stride,
                            const int32_t* lengths, void* k, void* v, int32_t* status, void* stream) {
    if (const int rc = check_cache(cache)) return rc;
    if (!table || !lengths || !k || !v) return HTREE_E_NULL;
    if (B <= 0 || M <= 0 || T <= 0 || table_stride < M) return HTREE_E_SHAPE;
    if (B > 65535 || (int64_t)B * T >= (int64_t(1) << 31)) return HTREE_E_UNSUPPORTED;
    if (!cache_aligned(k) || !cache_aligned(v)) return HTREE_E_ALIGN;
    MoveParams p;
    fill_move(p, *cache, status);
    p.ok = (char*)k; p.ov = (char*)v; p.table = table; p.table_stride = table_stride; p.lengths = lengths; p.n = T;
    p.tokens = (int64_t)B * T; p.per_row = FastDiv((uint32_t)T);
    const int64_t room = (int64_t)M * cache->page_size;
    p.room = (int32_t)(room < 0x7fffffff ? room : 0x7fffffff);
    return launch_chained(cache_gather_kernel, move_grid(p), dim3(256), 0, (cudaStream_t)stream, p);
}

}  // extern "C"
