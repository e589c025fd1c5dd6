// Eviction from a gather cache by the attention that each token has gathered.
//
// Per sequence and key head, the `keep` slots to stay are the first `sinks`, the last `recent` and the ones of the
// largest mass between them.  select_kernel, one block a (sequence, key head), finds the smallest kept mass by radix
// selection (three histograms of 11, 11 and 10 bits of an order-preserving integer key; the keys stay in shared
// memory, so the mass is read once) and writes the kept slots in ascending order.  move_kernel then moves the rows.
//
// In place, rank r comes from slot s >= r.  A block owns one pool's rows of one (sequence, key head), or a slice of
// their columns, and goes through the ranks in ascending chunks: all loads of a chunk, a barrier, all stores.  Stores
// of ranks [a, b) reach slots below b, which later ranks no longer read, so nothing is overwritten early.  The same
// order serves fresh pages.  Rows that stay where they are cost nothing.  While a chunk's rows are on their way, the
// next chunk's places are looked up (kept slot, page, row: three dependent loads), one thread a row.
//
// The move is bound by memory traffic (16 D + 4 bytes read and written per kept token and key head): 32 sequences of
// 8000 slots down to 4000, 4 key heads of 128: 183 us, 5.8 TB/s of rows of 256 bytes, 0.88 of a plain copy's rate; the
// selection before it 22 us.  (A row's address as one 64-bit product from the block's own pointer: formed from row, head
// and piece each time, the same loop took 225.)  Two sequences of 700 down to 333 take 9 and 4 us, bound by the latency of the passes.
#include <algorithm>

#include "att3_abi_internal.h"
#include "serve_common.cuh"

namespace {

constexpr int SEL_THREADS = 1024;
constexpr int BINS = 2048;
constexpr int SEL_SMEM_KEYS = 49152;        // 192 KB of keys; longer sequences read the mass again in every pass
constexpr int MOVE_THREADS = 256;
constexpr int MOVE_UNROLL = 8;              // 16-byte pieces a thread has in flight

struct Params {
    uint4* pool[4];
    float* mass;
    serve::Pages src, dst;
    const int* lengths;
    int* new_lengths;
    int* kept;
    int B, Hkv, keep, sinks, recent;
    int row16;              // 16-byte pieces of a row
    int slices;             // blocks that share a row's pieces
    int cached;             // keys fit in shared memory
    int* status;
};

// Larger mass, larger key; NaN above everything, both zeros alike.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Pair { int a, b; };

// Exclusive sums over the block of two counts a thread, and their totals.
__device__ __forceinline__ Pair block_scan(int a, int b, int2* warp_sums, Pair* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int xa = a, xb = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int ya = __shfl_up_sync(0xFFFFFFFFu, xa, o), yb = __shfl_up_sync(0xFFFFFFFFu, xb, o);
        if (lane >= o) { xa += ya; xb += yb; }
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = make_int2(xa, xb);
    __syncthreads();
    int ba = 0, bb = 0, ta = 0, tb = 0;
#pragma unroll
    for (int w = 0; w < SEL_THREADS / 32; ++w) {
        const int2 s = warp_sums[w];
        if (w < warp) { ba += s.x; bb += s.y; }
        ta += s.x;
        tb += s.y;
    }
    *total = Pair{ta, tb};
    return Pair{ba + xa - a, bb + xb - b};
}

__global__ void __launch_bounds__(SEL_THREADS) select_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[BINS];
    __shared__ int2 warp_sums[SEL_THREADS / 32];
    __shared__ int chosen[2];
    serve::wait_for_previous_kernel();
    const int h = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv, tid = threadIdx.x;
    const int n = p.src.length(p.lengths, b, p.status, tid == 0 && h == 0);
    int* kept = p.kept + static_cast<long long>(blockIdx.x) * p.keep;
    const int left = min(n, p.keep);
    if (h == 0 && tid == 0) p.new_lengths[b] = left;
    // Counts go up to 2^31 - 1, a step beyond them would be negative: loops over ranks and slots count unsigned.
    const unsigned keep = p.keep;
    for (unsigned r = left + tid; r < keep; r += SEL_THREADS) kept[r] = -1;
    if (n <= p.keep) {
        for (unsigned r = tid; r < static_cast<unsigned>(n); r += SEL_THREADS) kept[r] = r;
        return;
    }
    // here sinks + recent <= keep < n: the held ends do not meet
    const int first = p.sinks, want = p.keep - p.sinks - p.recent;
    const unsigned M = n - p.sinks - p.recent, recent = p.recent;
    for (unsigned r = tid; r < static_cast<unsigned>(p.sinks); r += SEL_THREADS) kept[r] = r;
    for (unsigned r = tid; r < recent; r += SEL_THREADS) kept[keep - recent + r] = n - recent + r;
    if (want == 0) return;

    auto fetch = [&](unsigned i) -> uint32_t {
        const int row = p.src.row(b, first + i);
        if (row < 0) { serve::report(p.status, serve::ST_PAGE); return 0u; }
        return order_key(p.mass[static_cast<long long>(row) * p.Hkv + h]);
    };
    auto key_of = [&](unsigned i) -> uint32_t { return p.cached ? keys[i] : fetch(i); };
    if (p.cached) {
#pragma unroll 4
        for (unsigned i = tid; i < M; i += SEL_THREADS) keys[i] = fetch(i);
    }

    // `prefix`: the leading bits of the want-th largest key; `more`: how many of the keys that share them still count
    uint32_t prefix = 0, done = 0;
    int more = want;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < BINS; i += SEL_THREADS) hist[i] = 0;
        __syncthreads();
        for (unsigned i = tid; i < M; i += SEL_THREADS) {
            const uint32_t k = key_of(i);
            if ((k & done) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1u)], 1);
        }
        __syncthreads();
        // thread t looks at the bins from the top: 2t and 2t + 1 of BINS - 1 - bin
        const int hi = BINS - 1 - 2 * tid;
        const int c0 = hist[hi], c1 = hist[hi - 1];
        Pair total;
        const Pair before = block_scan(c0 + c1, 0, warp_sums, &total);
        if (before.a < more && more <= before.a + c0 + c1) {
            const bool up = more <= before.a + c0;
            chosen[0] = up ? hi : hi - 1;
            chosen[1] = more - before.a - (up ? 0 : c0);
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(chosen[0]) << shift;
        done |= ((1u << bits) - 1u) << shift;
        more = chosen[1];
    }
    // keys above `prefix` stay, and the first `more` that equal it.  Each thread ranks a run of neighbouring slots.
    const unsigned run = (M + SEL_THREADS - 1) / SEL_THREADS, lo = min(tid * run, M), hi = min(lo + run, M);
    int above = 0, equal = 0;
    for (unsigned i = lo; i < hi; ++i) {
        const uint32_t k = key_of(i);
        above += k > prefix;
        equal += k == prefix;
    }
    Pair total;
    const Pair before = block_scan(above, equal, warp_sums, &total);
    int ahead = before.a, same = before.b;
    for (unsigned i = lo; i < hi; ++i) {
        const uint32_t k = key_of(i);
        if (k > prefix || (k == prefix && same < more)) kept[p.sinks + ahead + min(same, more)] = first + i;
        ahead += k > prefix;
        same += k == prefix;
    }
}

// blockIdx.x: (sequence, key head); blockIdx.y: pool * slices + slice, the last one the mass.
__global__ void __launch_bounds__(MOVE_THREADS, 4) move_kernel(const __grid_constant__ Params p) {
    constexpr int MOST = MOVE_THREADS * MOVE_UNROLL;                   // rows of a chunk: that many of masses, fewer of pools
    __shared__ int from[2][MOST / 2], to[2][MOST / 2];
    serve::wait_for_previous_kernel();
    const int h = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv;
    const int n = p.src.length(p.lengths, b, p.status, false);
    const unsigned left = min(n, p.keep);                              // unsigned: a chunk's end may pass 2^31
    const int* kept = p.kept + static_cast<long long>(blockIdx.x) * p.keep;
    const bool is_mass = static_cast<int>(blockIdx.y) == 4 * p.slices;
    const int width = is_mass ? 2 : p.row16 / p.slices;                // threads a row (two share a mass: the first moves it)
    const int at = is_mass ? 0 : (blockIdx.y % p.slices) * width + threadIdx.x % width;
    const int rows = MOVE_THREADS / width, mine = threadIdx.x / width, chunk = rows * MOVE_UNROLL;
    const bool idle = is_mass && threadIdx.x % width != 0;
    uint4* pool = is_mass ? nullptr : p.pool[blockIdx.y / p.slices] + static_cast<long long>(h) * p.row16 + at;
    const unsigned pitch = static_cast<unsigned>(p.Hkv) * p.row16;
    float* mass = p.mass + h;
    // places of a chunk's rows: source row, target row; the source is -1 where nothing moves
    auto look = [&](unsigned base, int buf) {
        for (int i = threadIdx.x; i < chunk && base + i < left; i += MOVE_THREADS) {
            int s = p.src.row(b, kept[base + i]);
            const int d = p.dst.row(b, base + i);
            if (s < 0 || d < 0) { serve::report(p.status, serve::ST_PAGE); s = -1; }
            from[buf][i] = s == d ? -1 : s;
            to[buf][i] = d;
        }
    };
    look(0, 0);
    __syncthreads();
    int buf = 0;
    for (unsigned base = 0; base < left; base += chunk, buf ^= 1) {
        uint4 v[MOVE_UNROLL];
#pragma unroll
        for (int u = 0; u < MOVE_UNROLL; ++u) {
            const int i = u * rows + mine;
            if (idle || base + i >= left) continue;
            const int s = from[buf][i];
            if (s < 0) continue;
            if (is_mass) v[u].x = __float_as_uint(mass[static_cast<long long>(s) * p.Hkv]);
            else v[u] = pool[static_cast<unsigned long long>(static_cast<unsigned>(s)) * pitch];
        }
        look(base + chunk, buf ^ 1);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < MOVE_UNROLL; ++u) {
            const int i = u * rows + mine;
            if (idle || base + i >= left || from[buf][i] < 0) continue;
            if (is_mass) mass[static_cast<long long>(to[buf][i]) * p.Hkv] = __uint_as_float(v[u].x);
            else pool[static_cast<unsigned long long>(static_cast<unsigned>(to[buf][i])) * pitch] = v[u];
        }
        __syncthreads();                                               // the buffer is looked up into again
    }
}

}  // namespace

namespace att3 {

int check_gather_pages(const att3_gather_pages* g, const char* who) {
    if (!g || !g->table) return set_error(ATT3_ERR_INVALID, "%s: null page table", who);
    if (g->page_size < 1 || g->pages < 1 || g->per_sequence < 1)
        return set_error(ATT3_ERR_INVALID, "%s: page size, pages and table width must be positive", who);
    constexpr int64_t most = 0x7FFFFFFFll;
    if (g->pages > most || g->page_size > most || g->per_sequence > most || g->pages * g->page_size > most || g->per_sequence * g->page_size > most)
        return set_error(ATT3_ERR_INVALID, "%s: a pool or a sequence of more than 2^31 - 1 slots", who);
    return ATT3_OK;
}

}  // namespace att3

extern "C" int att3_gather_cache_evict(void* R, void* S, void* Vr, void* Vs, float* mass, const att3_gather_pages* pages,
                                       const att3_gather_pages* out, const int32_t* lengths, int32_t* new_lengths,
                                       int32_t* kept, int B, int Hkv, int D, int keep, int sinks, int recent, void* stream) {
    const char* who = "att3_gather_cache_evict";
    if (B < 0 || Hkv < 1) return att3::set_error(ATT3_ERR_INVALID, "%s: empty head dimension", who);
    if (D != 16 && D != 32 && D != 64 && D != 128)
        return att3::set_error(ATT3_ERR_INVALID, "%s: head dim must be 16, 32, 64 or 128, got %d", who, D);
    if (keep < 1 || sinks < 0 || recent < 0 || static_cast<long long>(sinks) + recent > keep)
        return att3::set_error(ATT3_ERR_INVALID, "%s: sinks + recent must fit in keep >= 1, got %d + %d in %d", who, sinks, recent, keep);
    if (B == 0) return ATT3_OK;
    if (static_cast<long long>(B) * Hkv > 0x7FFFFFFFll) return att3::set_error(ATT3_ERR_INVALID, "%s: too many heads", who);
    if (int rc = att3::check_gather_pages(pages, who)) return rc;
    if (int rc = att3::check_gather_pages(out, who)) return rc;
    if (out->per_sequence * out->page_size < std::min<long long>(keep, pages->per_sequence * pages->page_size))
        return att3::set_error(ATT3_ERR_INVALID, "%s: the output table has no room for %d slots", who, keep);
    if (out->page_size != pages->page_size || out->pages != pages->pages)
        return att3::set_error(ATT3_ERR_INVALID, "%s: both tables must name pages of the same pools", who);
    if (!R || !S || !Vr || !Vs || !mass || !lengths || !new_lengths || !kept) return att3::set_error(ATT3_ERR_INVALID, "%s: null tensor", who);
    void* pools[4] = {R, S, Vr, Vs};
    for (void* q : pools)
        if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return att3::set_error(ATT3_ERR_INVALID, "%s: pools must be 16-byte aligned", who);
    if (!att3::require_sm100(who)) return ATT3_ERR_UNSUPPORTED;
    Params p = {};
    for (int k = 0; k < 4; ++k) p.pool[k] = static_cast<uint4*>(pools[k]);
    p.mass = mass;
    auto view = [](const att3_gather_pages* g) {
        return serve::make_pages(g->table, g->table_stride, g->per_sequence, g->pages, g->page_size);
    };
    p.src = view(pages);
    p.dst = view(out);
    p.lengths = lengths; p.new_lengths = new_lengths; p.kept = kept;
    p.B = B; p.Hkv = Hkv; p.keep = keep; p.sinks = sinks; p.recent = recent;
    p.row16 = D / 8;
    const long long most = pages->per_sequence * pages->page_size;
    p.cached = most <= SEL_SMEM_KEYS;
    if (!(p.status = att3::serve_status_ptr())) return att3::set_error(ATT3_ERR_CUDA, "%s: status word not resolvable", who);
    // whole rows a block when there are sequences and heads enough for two blocks an SM, else slices of their columns,
    // no thinner than a 32-byte sector
    p.slices = 1;
    while (p.slices * 2 <= p.row16 / 2 && static_cast<long long>(B) * Hkv * 4 * p.slices < 2ll * att3::sm_count()) p.slices *= 2;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int smem = p.cached ? static_cast<int>(most) * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_SMEM_KEYS * 4);
    if (e != cudaSuccess) return att3::set_cuda_error(e, who);
    att3::count_launch(4, 2);
    const att3::TimedLaunch timed(att3::K_SERVE, st);
    e = serve::launch_early(select_kernel, dim3(B * Hkv), dim3(SEL_THREADS), smem, st, p);
    if (e == cudaSuccess) e = serve::launch_early(move_kernel, dim3(B * Hkv, 4 * p.slices + 1), dim3(MOVE_THREADS), 0, st, p);
    return e == cudaSuccess ? ATT3_OK : att3::set_cuda_error(e, who);
}
